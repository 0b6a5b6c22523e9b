"""The kernels that keep activations in 8 bits, against 64-bit definitions (needs a B200).

Tolerances count roundings: 2^-8 of a bf16 result; fp32 arithmetic of a row (chains of at most 64 additions) 2^-17 of the operands;
exponentials and quotients of the fast kind 2^-16."""
import pytest
import torch

import act8_oracle as O

pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "int8"]
BF = 2.0 ** -8 + 2.0 ** -15


@pytest.fixture(scope="module", autouse=True)
def lib():
    from odysseus_transformer_b200.ops import native
    native.set_backend("fused")
    return native.lib()


@pytest.fixture(scope="module")
def F():
    from odysseus_transformer_b200.ops import functional
    return functional


@pytest.fixture(scope="module")
def R():
    from odysseus_transformer_b200.ops import torch_ref
    return torch_ref


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(T, n, seed=0, scale=1.0):
    x = torch.randn(T, n, generator=_gen(seed), device="cuda") * scale
    x[:, ::97] *= 30.0
    return x.bfloat16()


def _tiny(a, b=None):
    """Sigmoids below 2^-126 count as zero: a product with one is off by at most the other factors times 2^-126; and results below
    bf16's normal range are rounded to multiples of 2^-133."""
    return (a.double() if b is None else a.double() * b.double()).abs() * 2.0 ** -126 + 2.0 ** -133


def _values(kept):
    return kept.data.double() * O.spread(kept.scale, kept.data.shape[1])


def _same_codes(kept, want, what=""):
    """Codes and scales of two sides that compute them by the same roundings (``want`` on any device)."""
    data, scale = (t.to(kept.data.device) for t in want)
    finite = torch.isfinite(scale)
    assert torch.equal(finite, torch.isfinite(kept.scale)), what
    assert torch.equal(kept.scale[finite], scale[finite]), what
    ok = finite.repeat_interleave(128, 1)[:, :data.shape[1]]
    assert torch.equal(kept.data.float()[ok], data.float()[ok]), what


# one column group and less, ragged groups, several column tiles, rows that are whole 32-byte pieces and rows that are not
WIDTHS = [8, 16, 120, 128, 136, 256, 688, 1032, 4096, 4104, 11008]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("T", [1, 2, 37, 300])
def test_pack_and_unpack(F, R, fmt, T, n):
    x = _rows(T, n, seed=T * 7 + n)
    x[T // 2, : n // 2] = 0
    kept = F.pack8(x, fmt)
    _same_codes(kept, R.pack8(x.cpu(), fmt))
    back = F.unpack8(kept)
    assert back.dtype == x.dtype and torch.equal(back, _values(kept).float().bfloat16())
    if fmt == "e4m3" and T * n < 20000:
        codes, scales = O.keep(x.cpu(), fmt)
        assert torch.equal(back.double().cpu(), codes * scales)


@pytest.mark.parametrize("fmt", FMTS)
def test_pack_edges(F, R, fmt):
    x = torch.zeros(9, 304, device="cuda", dtype=torch.bfloat16)
    x[1, 5] = 2.0 ** -101
    x[2] = 2.0 ** -100
    x[3, 130], x[3, 260], x[3, 7] = float("inf"), float("nan"), 3.0
    x[4, :128] = torch.finfo(torch.bfloat16).min
    x[4, 3] = torch.finfo(torch.bfloat16).max
    x[5, 0], x[5, 1] = 448.0, 2.0 ** -9
    x[6, ::2], x[6, 1::2] = 1.75 * 2.0 ** 127, 1.0
    x[7] = 2.0 ** -133                                  # the type's smallest
    x[8, 303] = float("-inf")
    kept = F.pack8(x, fmt)
    _same_codes(kept, R.pack8(x.cpu(), fmt))
    y = F.unpack8(kept).cpu()
    want = R.unpack8(*R.pack8(x.cpu(), fmt), None, torch.bfloat16)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(), want.nan_to_num())
    assert y[3, 128:].isnan().all() and y[8, 256:].isnan().all() and not y[3, :128].isnan().any()
    assert not y.isinf().any()


@pytest.mark.parametrize("e", [-107, -3, 0, 120])
def test_int8_codes_on_their_borders(F, e):
    """The nearest code, and of two as near the even one, from every kernel that makes codes; in accesses of 32 and of 16 bytes."""
    x, codes = (t.cuda() for t in O.borders())
    x = torch.ldexp(x, torch.tensor(e, device="cuda")).bfloat16()
    wide, want = torch.cat([x, x.flip(0)], 1), torch.cat([codes, codes.flip(0)], 1)
    ragged = torch.cat([wide, x.new_zeros(len(x), 8)], 1)
    for t, n in ((wide, 256), (ragged, 264)):
        assert torch.equal(F.pack8(t, "int8").data[:, :256].long(), want)
        assert torch.equal(F.swiglu8(torch.cat([t, t], 1), "int8")[1].data.view(-1, 2, n)[..., :256].long(), want.unsqueeze(1).expand(-1, 2, -1))
        w = torch.ones(n, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(F.rmsnorm8(t, w, 1e-5, "int8")[1].data[:, :256].long(), want)
        s, _, kept = F.add_rmsnorm8(t, torch.zeros_like(t), w, 1e-5, "int8")
        assert torch.equal(s, t) and torch.equal(kept.data[:, :256].long(), want)


def test_pack_of_views(F):
    """Rows that lie apart, other starts, other orders; and nothing beyond the tensor is written or read."""
    x = _rows(40, 2048, seed=3)
    for t in (x[:, 8:1032], x[:, 16:1040], x[::3, :512], x[1:, 4:132], x.t(), x[:, :1].expand(40, 64), x.view(8, 5, 2048), x[5]):
        a, b = F.pack8(t, "int8"), F.pack8(t.contiguous().clone(), "int8")
        assert torch.equal(a.data, b.data) and torch.equal(a.scale, b.scale)
        assert torch.equal(F.unpack8(a), F.unpack8(b)) and F.unpack8(a).shape == t.shape


def test_empty(F):
    for fmt in FMTS:
        x = torch.empty(0, 256, device="cuda", dtype=torch.bfloat16).requires_grad_()
        w = torch.ones(256, device="cuda", dtype=torch.bfloat16).requires_grad_()
        assert F.unpack8(F.pack8(x, fmt)).shape == x.shape
        s, y, kept = F.rmsnorm_keep8(x, w, 1e-5, fmt)
        dx, dw = torch.autograd.grad((s, y), (x, w), (torch.empty_like(s), torch.empty_like(y)))
        assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(dw)) and kept.restore().shape == x.shape
        h, kept = F.swiglu8(x, fmt)
        assert h.shape == (0, 128) and kept.restore().shape == h.shape
        assert torch.autograd.grad(h, x, torch.empty_like(h))[0].shape == x.shape


def test_refusals(F, lib):
    x, w = _rows(4, 64), torch.ones(64, device="cuda", dtype=torch.bfloat16)
    bad = [lambda: F.pack8(x[:, :60].contiguous()), lambda: F.rmsnorm8(x[:, :4].contiguous(), w[:4], 1e-5), lambda: F.swiglu8(x[:, :24].contiguous()),
           lambda: F.rmsnorm8(_rows(2, 16392), torch.ones(16392, device="cuda", dtype=torch.bfloat16), 1e-5),
           lambda: lib.pack8(x, "fp8"), lambda: lib.pack8(x.float(), "int8"), lambda: lib.unpack8(x, x, None)]
    k = F.pack8(x)
    bad += [lambda: lib.unpack8(k.data, k.scale[:2], None), lambda: lib.unpack8(k.data, k.scale.double(), None),
            lambda: lib.unpack8(k.data, k.scale, w[:32]), lambda: lib.unpack8(k.data, k.scale.cpu(), None),
            lambda: lib.unpack8(k.data[:, :32], k.scale, None), lambda: lib.swiglu8_restore(k.data, k.scale),
            lambda: lib.swiglu8_bwd(x, k.data, k.scale), lambda: lib.rmsnorm8_bwd(x[:2], k.data, k.scale, w, k.scale[:, 0]),
            lambda: lib.rmsnorm8_bwd(x, k.data, k.scale, w[:8], k.scale[:, 0].contiguous()), lambda: F.linear(x, w.view(1, 64), kept=F.pack8(x[:2]))]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [8, 120, 256, 688, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200, 16384])
@pytest.mark.parametrize("T,form", [(1, "add"), (37, "norm"), (700, "keep"), (700, "add")])
def test_norm(F, R, fmt, n, T, form):
    if T * n > 4 << 20:
        T = 301                                         # some blocks get two rows, others one
    x, delta, dy, ds = (_rows(T, n, seed=i + n, scale=s) for i, s in enumerate((1.0, 0.3, 0.1, 0.1)))
    w = (1 + 0.2 * torch.randn(n, generator=_gen(9), device="cuda")).bfloat16()
    x[T // 2] = 0
    if form == "add":
        delta[T // 2] = 0
    for t in (x, delta, w):
        t.requires_grad_()
    if form == "norm":
        (y, kept), s = F.rmsnorm8(x, w, 1e-5, fmt), x
    elif form == "keep":
        s, y, kept = F.rmsnorm_keep8(x, w, 1e-5, fmt)
    else:
        s, y, kept = F.add_rmsnorm8(x, delta, w, 1e-5, fmt)
    s0, w0 = s.detach(), w.detach()
    assert torch.equal(s0, x.detach() + delta.detach() if form == "add" else x.detach())
    want, xh, r = O.norm(s0, w0, 1e-5)
    assert ((y.double() - want).abs() <= want.abs() * BF).all()
    data, scale = R.pack8(s0.cpu(), fmt)
    assert torch.equal(kept.data.float(), data.cuda().float())
    assert ((kept.scale.double() - scale.cuda().double() * r).abs() <= scale.cuda().double() * r * 2.0 ** -17).all()
    got = _values(kept)
    back = kept.restore()
    assert ((back.double() - got * w0.double()).abs() <= (got * w0.double()).abs() * BF).all()
    outs, grads = ((y,), (dy,)) if form == "norm" else ((s, y), (ds, dy))
    dx, dw, *rest = torch.autograd.grad(outs, (x, w) if form != "add" else (x, w, delta), grads)
    wx, ww = O.norm_grad(dy, got, w0, r, None if form == "norm" else ds)
    g = (dy.double() * w0.double())
    tol = r * (g.abs() + got.abs() * (g * got).abs().mean(1, keepdim=True)) * 2.0 ** -17 + ds.double().abs() * 2.0 ** -22
    assert ((dx.double() - wx).abs() <= wx.abs() * BF + tol).all()
    # a block adds up to three rows in turn, the blocks' sums ten at a time and then 32
    assert ((dw.double() - ww).abs() <= ww.abs() * BF + (dy.double() * got).abs().sum(0) * 64 * 2.0 ** -24).all()
    if rest:
        assert torch.equal(rest[0], dx)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,T", [(8, 24001), (256, 24001), (1024, 6001), (1032, 6001), (2048, 3001), (2056, 4501), (4096, 3001), (4104, 3001), (8192, 1501),
                                 (8200, 1501), (16384, 1501)])
@pytest.mark.parametrize("form", ["norm", "keep"])
def test_norm_gradient_of_many_rows_a_block(F, fmt, n, T, form):
    """Blocks with ten rows and more: every slot of the ring of rows is used several times, and sums go over all of them."""
    x, dy, ds = (_rows(T, n, seed=i + n, scale=s) for i, s in enumerate((1.0, 0.1, 0.1)))
    w = (1 + 0.2 * torch.randn(n, generator=_gen(9), device="cuda")).bfloat16()
    for t in (x, w):
        t.requires_grad_()
    if form == "norm":
        (y, kept), s = F.rmsnorm8(x, w, 1e-5, fmt), x
    else:
        s, y, kept = F.rmsnorm_keep8(x, w, 1e-5, fmt)
    outs, grads = ((y,), (dy,)) if form == "norm" else ((s, y), (ds, dy))
    dx, dw = torch.autograd.grad(outs, (x, w), grads)
    w0, got = w.detach(), _values(kept)
    _, _, r = O.norm(x.detach(), w0, 1e-5)
    wx, ww = O.norm_grad(dy, got, w0, r, None if form == "norm" else ds)
    g = dy.double() * w0.double()
    tol = r * (g.abs() + got.abs() * (g * got).abs().mean(1, keepdim=True)) * 2.0 ** -17 + ds.double().abs() * 2.0 ** -22
    assert ((dx.double() - wx).abs() <= wx.abs() * BF + tol).all()
    # up to 14 rows in turn, up to 2368 blocks' sums in 32 shares of 74, and five halvings
    assert ((dw.double() - ww).abs() <= ww.abs() * BF + (dy.double() * got).abs().sum(0) * 96 * 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [8, 120, 128, 688, 1032, 2816, 11008])
@pytest.mark.parametrize("T", [1, 37, 200])
def test_swiglu(F, R, fmt, n, T):
    gu, dh = _rows(T, 2 * n, seed=n, scale=1.5), _rows(T, n, seed=n + 1, scale=0.1)
    gu[0, 0], gu[-1, n - 1] = -150.0, 150.0
    gu.requires_grad_()
    h, kept = F.swiglu8(gu, fmt)
    d = gu.detach()
    want = O.swiglu(d[:, :n], d[:, n:])
    assert ((h.double() - want).abs() <= want.abs() * (BF + 2.0 ** -16) + _tiny(d[:, :n].float(), d[:, n:].float())).all()
    (cg, sg), (cu, su) = R.pack8(d[:, :n].cpu(), fmt), R.pack8(d[:, n:].cpu(), fmt)
    _same_codes(kept, (torch.cat([cg.float(), cu.float()], 1), torch.cat([sg, su], 1))) if n % 128 == 0 else None
    groups = -(-n // 128)
    g, u = (kept.data[:, i * n:(i + 1) * n].double() * O.spread(kept.scale[:, i * groups:(i + 1) * groups], n) for i in (0, 1))
    for v, c, s in ((g, cg, sg), (u, cu, su)):
        assert torch.equal(v, c.cuda().double() * O.spread(s.cuda(), n))
    back, want = kept.restore(), O.swiglu(g, u)
    assert back.shape == h.shape and ((back.double() - want).abs() <= want.abs() * (BF + 2.0 ** -16) + _tiny(g, u)).all()
    (dgu,) = torch.autograd.grad(h, gu, dh)
    want = O.swiglu_grad(dh, g, u)
    size = dh.double().abs().repeat(1, 2) * torch.cat([u.abs() * (1 + g.abs()), g.abs()], 1)
    assert ((dgu.double() - want).abs() <= want.abs() * BF + size * torch.sigmoid(g).repeat(1, 2) * 2.0 ** -16 + _tiny(size)).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,T", [(128, 80001), (128, 120001), (688, 24001), (1032, 9001), (1032, 16001), (2816, 2401), (2824, 3601), (11008, 1001)])
def test_swiglu_of_many_rows_a_block(F, R, fmt, n, T):
    """Blocks that go on to second, third and fourth rows, the last of them with rows missing: 32, 5, 3 or one row at a time, in accesses
    of 32 and of 16 bytes, up to three blocks beside one another."""
    test_swiglu(F, R, fmt, n, T)


@pytest.mark.parametrize("fmt", FMTS)
def test_not_finite(F, R, fmt):
    """Infinities and NaN show in what depends on them and nowhere else."""
    x = _rows(6, 512, seed=1)
    x[1, 3], x[4, 500] = float("nan"), float("inf")
    w, dy = torch.ones(512, device="cuda", dtype=torch.bfloat16), _rows(6, 512, seed=2, scale=0.1)
    xr = x.clone().requires_grad_()
    y, kept = F.rmsnorm8(xr, w, 1e-5, fmt)
    (dx,) = torch.autograd.grad(y, xr, dy)
    back = kept.restore()
    for t in (y, back, dx):
        assert torch.isfinite(t[[0, 2, 3, 5]]).all()
        assert t[1].isnan().all() or t is y and t[1, 3].isnan()
    assert back[4, 384:].isnan().all() and dx[4].isnan().all()
    gu = x.clone().requires_grad_()
    h, kept = F.swiglu8(gu, fmt)
    (dgu,) = torch.autograd.grad(h, gu, dy[:, :256].contiguous())
    back = kept.restore()
    for t in (back, dgu, h):
        assert torch.isfinite(t[[0, 2, 3, 5]]).all()
    plain = torch.nn.functional.silu(x[:, :256].float()) * x[:, 256:].float()
    for bad in (torch.isnan, torch.isinf):
        assert torch.equal(bad(h), bad(plain))
    ends = torch.tensor([[float("inf"), 1.0] * 4 + [2.0, 1.0] * 4, [-200.0, -1.0] * 4 + [-3e38, 2.0] * 4], device="cuda", dtype=torch.bfloat16)
    assert torch.equal(F.swiglu8(ends, fmt)[0], torch.tensor([[float("inf"), 0.73105858] * 4, [0.0, -0.53788284] * 4], device="cuda").bfloat16())
    assert back[1, :128].isnan().all() and torch.isfinite(back[1, 128:]).all()
    assert back[4, 128:].isnan().all() and torch.isfinite(back[4, :128]).all()
    assert dgu[1, :128].isnan().all() and dgu[1, 256:384].isnan().all()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_with_kept_input(F, fmt):
    x, w, dy = _rows(301, 264).requires_grad_(), _rows(136, 264, seed=1, scale=0.02).requires_grad_(), _rows(301, 136, seed=2, scale=0.1)
    kept = F.pack8(x, fmt)
    y = F.linear(x, w, kept=kept)
    assert torch.equal(y, F.linear(x, w))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx, F.gemm_nn(dy, w.detach())) and torch.equal(dw, F.gemm_tn(dy, kept.restore()))


def test_shapes_and_gradients_of_all_kinds(F):
    """Leading dims, inputs that need no gradient, expanded gradients, gradients of one output, second derivatives refused."""
    x, w = _rows(12, 256, seed=1).view(3, 4, 256), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    flat = x.view(12, 256)
    a, b = x.clone().requires_grad_(), flat.clone().requires_grad_()
    for leaf in (a, b):
        s, y, kept = F.rmsnorm_keep8(leaf, w, 1e-5)
        h, kept_h = F.swiglu8(y)
        z = F.linear(h, _rows(64, 128, seed=2), kept=kept_h)
        assert s.shape == y.shape == kept.restore().shape == leaf.shape and h.shape == kept_h.restore().shape and z.shape == (*leaf.shape[:-1], 64)
        (s.sum() + z.sum()).backward()                   # an expanded gradient
    assert torch.equal(a.grad.view(12, 256), b.grad)
    c, wr = flat.clone().requires_grad_(), w.clone().requires_grad_()
    s, y, _ = F.rmsnorm_keep8(c, wr, 1e-5)
    one = torch.ones_like(s)
    ds = torch.autograd.grad(s, (c, wr), one, retain_graph=True, allow_unused=True)
    assert torch.equal(ds[0], one) and ds[1] is None
    dy = torch.autograd.grad(y, (c, wr), one, retain_graph=True)
    both = torch.autograd.grad((s, y), (c, wr), (one, one), retain_graph=True)
    assert torch.equal(both[1], dy[1]) and ((both[0].double() - 1 - dy[0].double()).abs() <= both[0].double().abs() * 2.0 ** -8 + dy[0].double().abs() * 2.0 ** -8).all()
    (dw,) = torch.autograd.grad(F.rmsnorm8(flat, wr, 1e-5)[0], wr, one)
    assert torch.equal(dw, dy[1])
    (again,) = torch.autograd.grad(y, c, one, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        again.sum().backward()
    for f in (lambda: F.swiglu8(c)[0], lambda: F.linear(c, _rows(8, 256), kept=F.pack8(c))):
        (again,) = torch.autograd.grad(f().sum(), c, create_graph=True)
        assert torch.equal(again, torch.autograd.grad(f().sum(), c)[0])
        with pytest.raises(RuntimeError, match="differentiated again"):
            (again * again).sum().backward()
    with torch.no_grad():
        assert F.rmsnorm8(c, wr, 1e-5)[0].grad_fn is None and F.swiglu8(c)[0].grad_fn is None
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: F.rmsnorm8(t, w, 1e-5)[0])(x)
    y = F.rmsnorm8(c, wr, 1e-5)[0]
    with torch.no_grad():
        wr.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(one)


def test_norm_gradients_that_are_delivered(F):
    """The weight gradient as the optimizer's buffer wants it: written, added, converted, and left alone for a frozen weight."""
    x, dy = _rows(40, 256), _rows(40, 256, seed=1, scale=0.1)
    w = torch.nn.Parameter(torch.ones(256, device="cuda", dtype=torch.bfloat16))
    F.rmsnorm8(x, w, 1e-5)[0].backward(dy)
    want = w.grad.clone()
    for dtype in (torch.bfloat16, torch.float32):
        w.grad, w.main_grad, w._grad_written = None, torch.full((256,), float("nan"), device="cuda", dtype=dtype), False
        F.rmsnorm8(x, w, 1e-5)[0].backward(dy)
        assert w.grad is None and w._grad_written and torch.equal(w.main_grad.bfloat16(), want)
        F.rmsnorm8(x, w, 1e-5)[0].backward(dy)
        assert torch.allclose(w.main_grad.float(), 2 * want.float(), rtol=2.0 ** -6)
    w._grad_written = False
    w.main_grad.fill_(7)
    w.requires_grad_(False)
    y = F.rmsnorm8(x.clone().requires_grad_(), w, 1e-5)[0]
    y.backward(dy)
    assert (w.main_grad == 7).all() and not w._grad_written


@pytest.mark.parametrize("fmt", FMTS)
def test_run_of_them(F, fmt):
    """A block as the model runs it, on a stream of its own, twice, with gradients where the optimizer reads them."""
    T, d, n = 130, 256, 688
    x, dy = _rows(T, d, seed=4).requires_grad_(), _rows(T, d, seed=5, scale=0.1)
    ws = [(1 + 0.1 * torch.randn(d, generator=_gen(6), device="cuda")).bfloat16(), _rows(2 * n, d, seed=7, scale=0.05), _rows(d, n, seed=8, scale=0.05)]
    ws = [torch.nn.Parameter(w) for w in ws]

    def run(grads=None):
        for w in ws:
            w.grad, w._grad_written = None, False
            if grads is not None:
                w.main_grad = grads[id(w)]
            elif hasattr(w, "main_grad"):
                del w.main_grad
        s, h, kept = F.rmsnorm_keep8(x, ws[0], 1e-5, fmt)
        p, kept_p = F.swiglu8(F.linear(h, ws[1], kept=kept), fmt)
        out = s + F.linear(p, ws[2], kept=kept_p)
        x.grad = None
        out.backward(dy)
        return [out.detach().clone(), x.grad.clone()] + [w.grad.clone() if grads is None else grads[id(w)].clone() for w in ws]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = run()
        b = run({id(w): torch.full_like(w, float("nan")) for w in ws})
    torch.cuda.current_stream().wait_stream(side)
    for t, u, v in zip(want, a, b):
        assert torch.equal(t, u) and torch.equal(t, v)


def test_saved_tensors_that_are_hooked(F):
    """Under a checkpoint, an offload to the host and hooks of a user's own, the nodes get back what they saved."""
    from torch.utils.checkpoint import checkpoint
    x, dy = _rows(33, 256, seed=4), _rows(33, 64, seed=5, scale=0.1)
    ws = [torch.nn.Parameter(t) for t in (torch.ones(256, device="cuda", dtype=torch.bfloat16), _rows(64, 128, seed=6, scale=0.05))]

    def block(a):
        _, h, kept = F.rmsnorm_keep8(a, ws[0], 1e-5)
        p, kept_p = F.swiglu8(F.linear(h, torch.eye(256, device="cuda", dtype=torch.bfloat16), kept=kept))
        return F.linear(p, ws[1], kept=kept_p)

    def run(how):
        leaf = x.clone().requires_grad_()
        return [t.clone() for t in torch.autograd.grad(how(leaf), (leaf, *ws), dy)]

    def offloaded(a):
        with torch.autograd.graph.save_on_cpu():
            return block(a)

    want = run(block)
    for how in (lambda a: checkpoint(block, a, use_reentrant=False), offloaded):
        assert all(torch.equal(g, w) for g, w in zip(run(how), want))
    back = F.unpack8(F.pack8(x, "int8")).requires_grad_()                    # what the recomputation sees
    want = torch.autograd.grad(block(back), (back, *ws), dy)
    assert all(torch.equal(g, w) for g, w in zip(run(lambda a: F.checkpoint8(block, (a,), fmt="int8")), want))


def test_starts_that_are_not_aligned(F):
    """Contiguous tensors that start on 2, 8 and 16 bytes: copied, in narrow accesses, as they are."""
    flat = torch.randn(40 * 256 + 64, generator=_gen(1), device="cuda").bfloat16()
    for start in (1, 4, 8, 16):
        x = flat[start:start + 40 * 256].view(40, 256)
        ref = x.clone()
        for fmt in FMTS:
            a, b = F.pack8(x, fmt), F.pack8(ref, fmt)
            assert torch.equal(a.data.float(), b.data.float()) and torch.equal(a.scale, b.scale)
            y, k = F.rmsnorm8(x, flat[start + 3:start + 259], 1e-5, fmt)
            y0, k0 = F.rmsnorm8(ref, flat[start + 3:start + 259].clone(), 1e-5, fmt)
            assert torch.equal(y, y0) and torch.equal(k.restore(), k0.restore())
            gu, gu0 = x.detach().requires_grad_(), ref.clone().requires_grad_()
            (h, k), (h0, k0) = F.swiglu8(gu, fmt), F.swiglu8(gu0, fmt)
            dh = flat[start + 5:start + 5 + 40 * 128].view(40, 128)
            assert torch.equal(h, h0) and torch.equal(k.restore(), k0.restore())
            assert torch.equal(torch.autograd.grad(h, gu, dh)[0], torch.autograd.grad(h0, gu0, dh.clone())[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_types_without_kernels(F, dtype):
    """Types that the kernels do not take go through the plain form, on the device."""
    x = _rows(5, 200, seed=1).to(dtype).requires_grad_()
    w = torch.ones(200, device="cuda", dtype=dtype, requires_grad=True)
    assert F.unpack8(F.pack8(x)).dtype == dtype
    s, y, kept = F.rmsnorm_keep8(x, w, 1e-5)
    z = F.linear(y, torch.ones(8, 200, device="cuda", dtype=dtype, requires_grad=True), kept=kept)
    h, _ = F.swiglu8(s)
    (z.sum() + h.sum()).backward()
    assert x.grad.dtype == dtype and torch.isfinite(x.grad).all() and torch.isfinite(w.grad).all()
    top = torch.finfo(dtype).max
    assert torch.isfinite(F.unpack8(F.pack8(torch.full((1, 8), top, device="cuda", dtype=dtype)))).all()


def test_captured_and_replayed(F):
    """Two captured graphs that share nothing with what runs between their replays."""
    x, w, dy = _rows(64, 512), torch.ones(512, device="cuda", dtype=torch.bfloat16), _rows(64, 512, seed=1, scale=0.1)

    def step(a):
        leaf = a.detach().requires_grad_()
        s, y, kept = F.rmsnorm_keep8(leaf, w, 1e-5)
        h, kept_h = F.swiglu8(y)
        (dx,) = torch.autograd.grad((s, h), leaf, (dy, dy[:, :256].contiguous()))
        return dx, kept.restore(), kept_h.restore(), F.unpack8(F.pack8(a, "int8"))

    ins = [x.clone(), _rows(64, 512, seed=9)]
    want = [[t.clone() for t in step(a)] for a in ins]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for a in ins:
            step(a)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for a in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(a))
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
        step(ins[1])
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    other = _rows(64, 512, seed=11)
    ins[0].copy_(other)
    graphs[0].replay()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], step(other)))


def test_launches_are_counted(F, lib):
    x, w = _rows(16, 256).requires_grad_(), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    lib.reset_launch_count()
    _, kept = F.rmsnorm8(x, w, 1e-5)
    kept.restore()
    F.unpack8(F.pack8(x))
    h, kept = F.swiglu8(x)
    kept.restore()
    assert lib.launch_count() == 6
    torch.autograd.grad(h, x, torch.ones_like(h))
    assert lib.launch_count() == 7


def test_offsets_past_32_bits(F, lib):
    """Over 2^31 values: the first and the last rows."""
    T, n = (1 << 19) + 3, 4096 + 16
    x = torch.zeros(T, n, device="cuda", dtype=torch.bfloat16)
    x[:2], x[-3:] = _rows(2, n, seed=1), _rows(3, n, seed=2)
    kept = F.pack8(x)
    back = F.unpack8(kept)
    for part in (slice(0, 2), slice(T - 3, T)):
        assert torch.equal(back[part], F.unpack8(F.pack8(x[part].clone())))
    del back, kept
    w = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y, kept = F.rmsnorm8(x, w, 1e-5)
    assert torch.equal(y[-3:], F.rmsnorm8(x[-3:].clone(), w, 1e-5)[0])
    back = kept.restore()
    assert torch.equal(back[-3:], F.rmsnorm8(x[-3:].clone(), w, 1e-5)[1].restore())
    del y
    dx, _ = lib.rmsnorm8_bwd(x, kept.data, kept.scale, w, torch.ones(T, device="cuda"))
    small = F.rmsnorm8(x[-3:].clone(), w, 1e-5)[1]
    assert torch.equal(dx[-3:], lib.rmsnorm8_bwd(x[-3:].clone(), small.data, small.scale, w, torch.ones(3, device="cuda"))[0])


def test_swiglu_offsets_past_32_bits(F):
    T, n = (1 << 19) + 3, 2048 + 8
    gu = torch.zeros(T, 2 * n, device="cuda", dtype=torch.bfloat16)
    gu[-3:] = _rows(3, 2 * n, seed=2)
    small = gu[-3:].clone().requires_grad_()
    h, kept = F.swiglu8(gu.requires_grad_())
    h3, kept3 = F.swiglu8(small)
    assert torch.equal(h[-3:], h3) and torch.equal(kept.restore()[-3:], kept3.restore())
    dh = torch.zeros_like(h)
    dh[-3:] = _rows(3, n, seed=3)
    assert torch.equal(torch.autograd.grad(h, gu, dh)[0][-3:], torch.autograd.grad(h3, small, dh[-3:].clone())[0])


def test_library_backend(F, R):
    """The plain forms on the device keep the same codes, and either side restores what the other kept."""
    from odysseus_transformer_b200.ops import native
    x, w, dy = _rows(30, 400, seed=1), torch.ones(400, device="cuda", dtype=torch.bfloat16), _rows(30, 400, seed=2, scale=0.1)
    out = {}
    for backend in ("library", "fused"):
        native.set_backend(backend)
        try:
            leaf = x.clone().requires_grad_()
            s, y, kept = F.rmsnorm_keep8(leaf, w, 1e-5)
            (dx,) = torch.autograd.grad((s, y), leaf, (dy, dy))
            out[backend] = (F.pack8(x, "int8"), kept, dx, F.swiglu8(x)[1])
        finally:
            native.set_backend("fused")
    a, b = out["library"], out["fused"]
    for i in (0, 1, 3):
        assert torch.equal(a[i].data.float(), b[i].data.float())
        assert ((a[i].restore().float() - b[i].restore().float()).abs() <= b[i].restore().float().abs() * 2.0 ** -7).all()
    assert torch.equal(a[0].restore(), b[0].restore())
    assert ((a[2].float() - b[2].float()).abs() <= b[2].float().abs() * 2.0 ** -7 + dy.float().abs() * 2.0 ** -7).all()


def test_inference_mode(F):
    x, w = _rows(9, 256), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    want = [F.rmsnorm8(x, w, 1e-5)[0], F.swiglu8(x)[0], F.unpack8(F.pack8(x)), F.linear(x, _rows(8, 256, seed=1))]
    with torch.inference_mode():
        y, kept = F.rmsnorm8(x, w, 1e-5)
        got = [y, F.swiglu8(x)[0], F.unpack8(F.pack8(x)), F.linear(x, _rows(8, 256, seed=1), kept=kept)]
        back = kept.restore()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(back, F.rmsnorm8(x, w, 1e-5)[1].restore())


def test_two_threads(F):
    """Two threads on streams of their own get what one gets."""
    import threading
    ins = [_rows(200, 512, seed=s) for s in (1, 2)]
    w, dy = torch.ones(512, device="cuda", dtype=torch.bfloat16), _rows(200, 512, seed=3, scale=0.1)

    def run(x):
        leaf = x.detach().requires_grad_()
        s, y, kept = F.rmsnorm_keep8(leaf, w, 1e-5, "int8")
        h, kept_h = F.swiglu8(y)
        return [kept.restore(), kept_h.restore(), *torch.autograd.grad((s, h), leaf, (dy, dy[:, :256].contiguous()))]

    want = [run(x) for x in ins]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = run(ins[i])
            stream.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and not any(t.is_alive() for t in threads)
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_tensors_left_over_from_a_transform(F):
    kept, x, w = [], _rows(4, 64), torch.ones(64, device="cuda", dtype=torch.bfloat16)

    def f(t):
        kept.append(t)
        return t.float().square().sum()

    torch.func.grad(f)(x)
    left = kept[0]
    assert torch.equal(F.rmsnorm8(left, w, 1e-5)[0], F.rmsnorm8(x, w, 1e-5)[0])
    assert torch.equal(F.swiglu8(left)[0], F.swiglu8(x)[0]) and torch.equal(F.unpack8(F.pack8(left)), F.unpack8(F.pack8(x)))
    assert torch.equal(F.linear(left, _rows(8, 64, seed=1), kept=F.pack8(x)), F.linear(x, _rows(8, 64, seed=1)))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            F.rmsnorm8(dual, w, 1e-5)


@pytest.mark.parametrize("mode", ["odysseus", "tpsp", "ulysses", "ring", "dp"])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_training_steps(mode, checkpoint):
    """A model with activations in 8 bits: the loss of the first step is the ordinary one's, every gradient is near the ordinary
    one's, and memory goes down.

    Gradients: a kept value is off by a rounding of at most 2^-4 of it, 2^-4 / sqrt(3) = 3.6 % in the mean square, and so is a
    weight gradient whose tokens' shares have nothing to do with one another, as with random tokens (shares that agree average
    the error out).  Two layers hold six kept tensors between the loss and the first weight: 3.6 % * sqrt(6) = 9 %, and not
    three times that."""
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import ParallelContext, set_context
    from odysseus_transformer_b200.train import Trainer
    cfg = get_model_config("small-gqa")
    ctx = ParallelContext(device=torch.device("cuda", 0), backend="fused")
    set_context(ctx)
    L = 1531
    batch = torch.randint(cfg.vocab_size, (1, L + 1), generator=torch.Generator().manual_seed(0)).pin_memory()
    got = {}
    for fmt in (None, "e4m3", "int8"):
        t = Trainer(cfg, mode, ctx, L, activations8=fmt, grad_checkpoint=checkpoint)
        s = t.shard_batch(batch)
        base = torch.cuda.memory_allocated()
        loss = t.model(s["local_input_ids"], s["local_position_ids"], labels=s["local_target_ids"], global_tokens=L)
        held = torch.cuda.memory_allocated() - base
        loss.backward()
        got[fmt] = (loss.detach().clone(), held, {k: p.main_grad.clone() for k, p in t.model.named_parameters()})
        t.optimizer.zero_grad()
        a, b = t.train_step(batch).item(), t.train_step(batch).item()
        assert torch.isfinite(torch.tensor([a, b])).all()
        t.check_status()
        del t, loss, s
    want = got[None]
    for fmt in FMTS:
        loss, held, grads = got[fmt]
        torch.testing.assert_close(loss, want[0], rtol=1e-5, atol=0)
        assert held < want[1]
        for k, g in want[2].items():
            assert (grads[k].float() - g.float()).norm() <= 0.25 * g.float().norm(), (fmt, k)
