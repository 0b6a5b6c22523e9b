"""Activations kept in 8 bits on the CPU path: what is kept, gradients against formulas and differences, refusals, and the model
in every mode.  Tolerances: fp32 arithmetic of a few operations is 2^-20 of the operands off at most, sums of up to 512 terms
2^-15."""
import math

import pytest
import torch

import act8_oracle as O
from dist_utils import run_distributed
from odysseus_transformer_b200.ops import functional as F
from odysseus_transformer_b200.ops import torch_ref as R

FMTS = ["e4m3", "int8"]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(T, n, seed=0, scale=1.0):
    g = _gen(seed)
    x = torch.randn(T, n, generator=g) * scale
    x[:, ::97] *= 30.0
    return x


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,n", [(1, 1), (3, 127), (2, 128), (5, 129), (4, 688), (0, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_values(fmt, T, n, dtype):
    x = _rows(T, n, seed=T + n).to(dtype)
    kept = F.pack8(x, fmt)
    assert kept.data.dtype == R.FORMATS8[fmt] and kept.data.shape == (T, n) and kept.scale.shape == (T, -(-n // 128))
    assert kept.nbytes == T * n + 4 * T * -(-n // 128)
    got = F.unpack8(kept)
    assert got.dtype == dtype and got.shape == x.shape
    codes, scales = O.keep(x, fmt)
    if fmt == "e4m3":                                   # powers of two: nothing but the code is rounded
        assert torch.equal(kept.data.double(), codes) and torch.equal(got.double(), codes * scales)
    else:                                               # at most half a step, and the type's rounding of the result
        half = scales * (0.5 + 127 * 2.0 ** -22) + x.double().abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -6)
        assert ((got.double() - x.double()).abs() <= half).all()


@pytest.mark.parametrize("e", [-107, -3, 0, 120])
def test_int8_codes_on_their_borders(e):
    """The nearest code, and of two as near the even one: half of a group's largest is 63.5 steps and becomes 64."""
    x, codes = O.borders()
    x = torch.ldexp(x, torch.tensor(e)).bfloat16()
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(F.pack8(x.to(dtype), "int8").data.long(), codes)
    a = torch.rand(500, 1, generator=_gen(1)) + 1       # of any fp32 number
    assert (F.pack8(torch.cat([a, a / 2, -a / 2], 1), "int8").data == torch.tensor([127, 64, -64])).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_kept_edges(fmt):
    x = torch.zeros(6, 300)
    x[1, 5] = 2.0 ** -101                               # below what has a scale
    x[2] = 2.0 ** -100
    x[3, 130], x[3, 260] = float("inf"), float("nan")
    x[3, 7] = 3.0
    x[4, :128] = torch.finfo(torch.bfloat16).min
    x[4, 3] = torch.finfo(torch.bfloat16).max
    x[5, 0], x[5, 1] = 448.0, 2.0 ** -9                 # the largest of e4m3 and its smallest
    y = F.unpack8(F.pack8(x, fmt))
    assert torch.equal(y[:2], torch.zeros(2, 300))
    assert torch.allclose(y[2], x[2], rtol=2.0 ** -20, atol=0)
    assert y[3, 128:].isnan().all()                     # both groups, whole
    assert y[3, 7] == pytest.approx(3.0, rel=2.0 ** -20) and y[3, :7].eq(0).all()
    assert torch.isfinite(y[4]).all() and torch.equal(y[4, 128:], x[4, 128:])   # e4m3 clips at 1.75 * 2^127, an eighth less
    assert torch.allclose(y[4], x[4], rtol=2.0 ** -3 if fmt == "e4m3" else 2.0 ** -20, atol=0)
    if fmt == "e4m3":
        assert torch.equal(y[5], x[5])


def test_kept_twice_is_kept_once():
    """e4m3: what was restored is kept as itself."""
    y = F.unpack8(F.pack8(_rows(7, 260).bfloat16()))
    assert torch.equal(F.unpack8(F.pack8(y)), y)


def test_shapes_strides_and_types():
    x = _rows(12, 96)
    for t in (x.view(3, 4, 96), x[:, 8:80], x.t(), x[::2], x[0], x[:, :1].expand(12, 50)):
        kept = F.pack8(t, "int8")
        assert kept.shape == t.shape and F.unpack8(kept).shape == t.shape
        assert torch.equal(F.unpack8(kept), F.unpack8(F.pack8(t.contiguous(), "int8")))


@pytest.mark.parametrize("call", [
    lambda x: F.pack8(x, "e5m2"), lambda x: F.pack8(torch.zeros(())), lambda x: F.pack8(torch.zeros(3, 0)),
    lambda x: F.pack8(torch.zeros(3, 4, dtype=torch.int64)), lambda x: F.rmsnorm8(x, torch.ones(3), 1e-5),
    lambda x: F.rmsnorm8(x, torch.ones(8), 1e-5, "fp8"), lambda x: F.add_rmsnorm8(x, x[:2], torch.ones(8), 1e-5),
    lambda x: F.swiglu8(x[:, :7]), lambda x: F.swiglu8(x, "int4"), lambda x: F.linear(x, torch.ones(4, 8), kept=F.pack8(x[:2])),
    lambda x: F.linear(x, torch.ones(4, 8), kept=F.pack8(x.double())), lambda x: F.checkpoint8(lambda a: a, (x,), fmt="int16")])
def test_refusals(call):
    with pytest.raises(ValueError):
        call(torch.randn(4, 8))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,n", [(1, 8), (5, 200), (37, 384)])
@pytest.mark.parametrize("form", ["norm", "keep", "add"])
def test_norm(fmt, T, n, form):
    x, delta, dy, ds = (_rows(T, n, seed=i + n) for i in range(4))
    w = 1 + 0.2 * torch.randn(n, generator=_gen(9))
    x.requires_grad_(), delta.requires_grad_(), w.requires_grad_()
    if form == "norm":
        y, kept = F.rmsnorm8(x, w, 1e-5, fmt)
        s = x
    elif form == "keep":
        s, y, kept = F.rmsnorm_keep8(x, w, 1e-5, fmt)
        assert torch.equal(s, x)
    else:
        s, y, kept = F.add_rmsnorm8(x, delta, w, 1e-5, fmt)
        assert torch.equal(s, x + delta)
    want, xh, r = O.norm(s.detach(), w.detach(), 1e-5)
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -17).all()
    codes, scales = O.keep(s.detach(), fmt)
    near = scales * r * 127 * 2.0 ** -20 if fmt == "int8" else 0
    got = kept.data.double() * O.spread(kept.scale, n)
    assert ((got - xh).abs() <= (codes * scales * r - xh).abs() + xh.abs() * 2.0 ** -17 + near).all()
    back = kept.restore()
    assert ((back.double() - got * w.detach().double()).abs() <= (got * w.detach().double()).abs() * 2.0 ** -20).all()
    outs, grads = ((y,), (dy,)) if form == "norm" else ((s, y), (ds, dy))
    ins = (x, w) if form != "add" else (x, w, delta)
    dx, dw, *rest = torch.autograd.grad(outs, ins, grads)
    wx, ww = O.norm_grad(dy, got, w.detach(), r, None if form == "norm" else ds)
    g = (dy * w.detach()).double()
    tol = r * (g.abs() + got.abs() * (g * got).abs().mean(1, keepdim=True)) * 2.0 ** -15 + ds.double().abs() * 2.0 ** -20
    assert ((dx.double() - wx).abs() <= tol).all()
    assert ((dw.double() - ww).abs() <= (dy.double() * got).abs().sum(0) * 2.0 ** -15).all()
    if rest:
        assert torch.equal(rest[0], dx)


def test_norm_gradient_of_one_output():
    x, w = _rows(4, 40).requires_grad_(), torch.ones(40, requires_grad=True)
    s, y, _ = F.rmsnorm_keep8(x, w, 1e-5)
    dx, dw = torch.autograd.grad(s, (x, w), torch.ones_like(s), retain_graph=True, allow_unused=True)
    assert torch.equal(dx, torch.ones_like(x)) and dw is None
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    both = torch.autograd.grad((s, y), (x, w), (torch.ones_like(s), torch.ones_like(y)))
    assert torch.allclose(both[0], dx + 1, rtol=2.0 ** -20, atol=2.0 ** -20) and torch.equal(both[1], dw)


def _representable(T, n, seed):
    """Values that e4m3 keeps exactly: few bits, and a group's sizes within its range."""
    g = _gen(seed)
    return torch.randint(-8, 9, (T, n), generator=g) * 0.25


def test_gradients_against_differences():
    """Where nothing is lost in keeping, the gradients are those of the forward pass: central differences in 64 bits."""
    T, n, h = 3, 136, 1e-5
    x, w, dy = _representable(T, n, 0), 1 + 0.1 * torch.randn(n, generator=_gen(1)), torch.randn(T, n, generator=_gen(2))
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = F.rmsnorm8(xr, wr, 1e-5)
    dx, dw = torch.autograd.grad(y, (xr, wr), dy)
    gu, dh = _representable(T, 2 * n, 3), torch.randn(T, n, generator=_gen(4))
    gr = gu.clone().requires_grad_()
    out, _ = F.swiglu8(gr)
    (dgu,) = torch.autograd.grad(out, gr, dh)
    f = lambda a, b: (O.norm(a, b, 1e-5)[0] * dy.double()).sum().item()     # noqa: E731
    s = lambda a: (O.swiglu(a[:, :n], a[:, n:]) * dh.double()).sum().item()     # noqa: E731
    for i, j in [(0, 0), (1, 127), (2, 128), (2, 135)]:
        e = torch.zeros(T, n, dtype=torch.float64)
        e[i, j] = h
        assert dx[i, j] == pytest.approx((f(x + e, w) - f(x - e, w)) / (2 * h), abs=1e-4)
        assert dw[j] == pytest.approx((f(x, w + e[i]) - f(x, w - e[i])) / (2 * h), abs=1e-4)
        for k in (j, n + j):
            e = torch.zeros(T, 2 * n, dtype=torch.float64)
            e[i, k] = h
            assert dgu[i, k] == pytest.approx((s(gu + e) - s(gu - e)) / (2 * h), abs=1e-4)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,n", [(1, 2), (3, 128), (6, 344)])
def test_swiglu(fmt, T, n):
    gu, dh = torch.randn(T, 2 * n, generator=_gen(n)) * 3, torch.randn(T, n, generator=_gen(n + 1))
    gu[0, 0], gu[-1, n - 1] = -150.0, 150.0             # exponentials at their ends
    gu.requires_grad_()
    h, kept = F.swiglu8(gu, fmt)
    d = gu.detach()
    want = O.swiglu(d[:, :n], d[:, n:])
    assert ((h.double() - want).abs() <= want.abs() * 2.0 ** -16 + 2.0 ** -120).all()
    groups = -(-n // 128)
    g, u = (kept.data[:, i * n:(i + 1) * n].double() * O.spread(kept.scale[:, i * groups:(i + 1) * groups], n) for i in (0, 1))
    for v, x in ((g, d[:, :n]), (u, d[:, n:])):
        codes, scales = O.keep(x, fmt)
        assert ((v - x.double()).abs() <= (codes * scales - x.double()).abs() + scales * 127 * 2.0 ** -20).all()
    back, want = kept.restore(), O.swiglu(g, u)
    assert back.shape == h.shape and ((back.double() - want).abs() <= want.abs() * 2.0 ** -16 + 2.0 ** -120).all()
    (dgu,) = torch.autograd.grad(h, gu, dh)
    want = O.swiglu_grad(dh, g, u)
    size = (dh.double().abs() * torch.sigmoid(g)).repeat(1, 2) * torch.cat([u.abs() * (1 + g.abs()), g.abs()], 1)
    assert ((dgu.double() - want).abs() <= size * 2.0 ** -16 + 2.0 ** -120).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_with_kept_input(fmt):
    x, w, dy = _rows(9, 150).requires_grad_(), torch.randn(20, 150, generator=_gen(3)).requires_grad_(), torch.randn(9, 20, generator=_gen(4))
    kept = F.pack8(x, fmt)
    y = F.linear(x, w, kept=kept)
    assert torch.equal(y, F.linear(x, w))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx, dy @ w) and torch.equal(dw, dy.t() @ kept.restore())


def test_run_of_them_in_a_block():
    """Norm, projection, SwiGLU, projection: what each keeps is what the next saves, and nothing of a kept tensor's own type."""
    T, d, n = 6, 64, 80
    x = _rows(T, d).requires_grad_()
    wn = torch.ones(d, requires_grad=True)
    wg, wd = (torch.randn(*s, generator=_gen(5)).mul_(0.1).requires_grad_() for s in ((2 * n, d), (d, n)))
    shapes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (shapes.append((tuple(t.shape), t.dtype)), t)[1], lambda t: t):
        s, h, kept = F.rmsnorm_keep8(x, wn, 1e-5)
        p, kept_p = F.swiglu8(F.linear(h, wg, kept=kept))
        out = s + F.linear(p, wd, kept=kept_p)
    assert not [s for s in shapes if s in [((T, d), torch.float32), ((T, n), torch.float32), ((T, 2 * n), torch.float32)]]
    dy = torch.randn(T, d, generator=_gen(6))
    dx, dwn, dwg, dwd = torch.autograd.grad(out, (x, wn, wg, wd), dy)
    dp = dy @ wd
    assert torch.equal(dwd, dy.t() @ kept_p.restore())
    dgu = R.swiglu8_bwd(dp, kept_p.data, kept_p.scale)
    assert torch.equal(dwg, dgu.t() @ kept.restore())
    r = (x.detach().square().mean(1) + 1e-5).rsqrt()
    wx, ww = R.rmsnorm8_bwd(dgu @ wg, kept.data, kept.scale, wn.detach(), r, dy)
    assert torch.allclose(dx, wx, rtol=1e-5, atol=1e-5) and torch.allclose(dwn, ww, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("fmt", FMTS)
def test_checkpoint(fmt):
    """The output is the function's; the gradients those of the function where its kept inputs have what their codes stand for."""
    x, y, w = _rows(5, 130).requires_grad_(), torch.randn(5, 130, generator=_gen(1)), torch.randn(7, 130, generator=_gen(2)).requires_grad_()
    calls = []

    def f(a, b, none, k, scale=1.0):
        calls.append(a.detach().clone())
        assert none is None
        return torch.tanh(a * k + b) @ w.t() * scale

    out = F.checkpoint8(f, (x, y, None), 0.5, fmt=fmt, scale=2.0)
    assert torch.equal(out, f(x, y, None, 0.5, 2.0)) and torch.equal(calls[0], x)
    dy = torch.randn(5, 7, generator=_gen(3))
    dx, dw = torch.autograd.grad(out, (x, w), dy, retain_graph=True)
    xs, ys = F.unpack8(F.pack8(x, fmt)).requires_grad_(), F.unpack8(F.pack8(y, fmt))
    wx, ww = torch.autograd.grad(f(xs, ys, None, 0.5, 2.0), (xs, w), dy)
    assert torch.equal(calls[2], xs) and torch.equal(dx, wx) and torch.equal(dw, ww)
    again = torch.autograd.grad(out, (x, w), dy)         # the codes are still there
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    with torch.no_grad():
        assert torch.equal(F.checkpoint8(f, (x, y, None), 0.5, fmt=fmt, scale=2.0), out)
    named = F.checkpoint8(lambda a, kept, function: a * kept + function, (x,), kept=2.0, function=1.0)     # names of its own
    assert torch.equal(named, x * 2 + 1)


def test_no_second_derivative():
    """A first derivative with a graph is the first derivative; what would differentiate it is refused and not taken as constant."""
    x, w = _rows(2, 16).requires_grad_(), torch.ones(4, 16, requires_grad=True)
    for f in (lambda: F.rmsnorm8(x, torch.ones(16), 1e-5)[0], lambda: F.swiglu8(x)[0], lambda: F.rmsnorm_keep8(x, torch.ones(16), 1e-5)[0]):
        (want,) = torch.autograd.grad(f().sum(), x)
        (dx,) = torch.autograd.grad(f().sum(), x, create_graph=True)
        assert torch.equal(dx, want) and dx.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            ((dx * dx).sum() + (x * x).sum()).backward()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(F.linear(x, w, kept=F.pack8(x)).sum(), x, create_graph=True)


def test_values_without_gradients():
    x, w = _rows(3, 24), torch.ones(24)
    with torch.no_grad():
        s, y, kept = F.rmsnorm_keep8(x, w, 1e-5)
        h, _ = F.swiglu8(x)
        z = F.linear(y, torch.ones(4, 24), kept=kept)
    assert torch.equal(y, F.rmsnorm(x, w, 1e-5)) and torch.equal(h, F.swiglu(x)) and torch.equal(s, x) and z.grad_fn is None


def _lossless(monkey=None):
    """Keeping without loss: the codes are the values.  What remains is who keeps what, and who reads it."""
    def pack8(x, fmt):
        return x.float().clone(), torch.ones(x.shape[0], -(-x.shape[1] // R.GROUP8))
    if monkey is not None:
        monkey.setattr(R, "pack8", pack8)
    else:
        R.pack8 = pack8


def _grads(rank, world, mode, cfg_name, L, U, RD, checkpoint, activations8, **kw):
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import init_parallel_context
    from odysseus_transformer_b200.parallel.apply import build_model, prepare_attn_inputs
    from odysseus_transformer_b200.utils.debug import export_hf_grads
    cfg = get_model_config(cfg_name)
    ctx = init_parallel_context(mode, U, RD, device=torch.device("cpu"), backend="library")
    model = build_model(cfg, mode, ctx, dtype=torch.float32, seed=0, activations8=activations8, **kw)
    if checkpoint:
        model.gradient_checkpointing_enable()
    batch = torch.randint(cfg.vocab_size, (1, L + 1), generator=_gen(0))
    s = prepare_attn_inputs(mode, batch[:, :-1], torch.arange(L).unsqueeze(0), batch[:, 1:], rank, world, "cpu", U, RD)
    loss = model(s["local_input_ids"], s["local_position_ids"], labels=s["local_target_ids"], global_tokens=L * (world if mode == "dp" else 1))
    loss.backward()
    return loss.detach(), export_hf_grads(model)


def _mode_lossless(rank, world, mode, cfg_name, L, U, RD, checkpoint):
    want = _grads(rank, world, mode, cfg_name, L, U, RD, checkpoint, None)
    _lossless()
    got = _grads(rank, world, mode, cfg_name, L, U, RD, checkpoint, "e4m3")
    assert torch.equal(got[0], want[0])
    for k, g in want[1].items():
        torch.testing.assert_close(got[1][k], g, rtol=1e-5, atol=1e-7, msg=lambda m: f"{mode} {k}: {m}")


@pytest.mark.parametrize("mode,checkpoint", [("odysseus", False), ("tpsp", False), ("ulysses", False), ("ring", False), ("dp", False),
                                             ("odysseus", True)])
def test_model_gradients_without_loss_world2(mode, checkpoint):
    """Restoring what was kept takes the place of saving in every mode: without loss in keeping, the gradients are the same."""
    run_distributed(_mode_lossless, 2, mode, "tiny-gqa", 64, 0, 1, checkpoint)


@pytest.mark.parametrize("mode", ["odysseus", "tpsp", None])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("checkpoint", [True, False])
def test_model_on_one_rank(mode, residual, checkpoint, monkeypatch):
    from odysseus_transformer_b200.mesh import ParallelContext
    from odysseus_transformer_b200.models.llama import LlamaForCausalLM
    from odysseus_transformer_b200.config import get_model_config
    monkeypatch.setitem(F._EPILOGUE_FUSION, "residual", residual)
    cfg = get_model_config("tiny")
    ids = torch.randint(cfg.vocab_size, (1, 33), generator=_gen(1))

    def step(activations8):
        m = LlamaForCausalLM(cfg, mode, ParallelContext(), activations8=activations8, use_zero3_linear=residual)
        m.init_weights(0)
        if checkpoint:
            m.gradient_checkpointing_enable()
        loss = m(ids[:, :-1], torch.arange(32).unsqueeze(0), labels=ids[:, 1:])
        loss.backward()
        return loss.detach(), {k: p.grad for k, p in m.named_parameters()}
    want, wg = step(None)
    for fmt in FMTS:
        loss, grads = step(fmt)
        assert torch.equal(loss, want) and all(torch.isfinite(g).all() for g in grads.values())
        assert any(not torch.equal(grads[k], wg[k]) for k in wg)
    _lossless(monkeypatch)
    _, grads = step("int8")
    for k, g in wg.items():
        torch.testing.assert_close(grads[k], g, rtol=1e-5, atol=1e-7, msg=lambda m: f"{k}: {m}")


@pytest.mark.parametrize("kw", [{}, {"bias": True}, {"sequence_parallel": False}, {"sequence_parallel": False, "bias": True}])
def test_linear_modules(kw):
    """Every form of the modules forms its weight gradient from what was kept."""
    from odysseus_transformer_b200.parallel.linear import ColumnParallelLinearAG, LinearZeRO3, RowParallelLinearRS
    x, dy = _rows(5, 24).requires_grad_(), torch.randn(5, 8, generator=_gen(1))
    mods = [ColumnParallelLinearAG(24, 8, None, **kw), RowParallelLinearRS(24, 8, None, **kw)] + ([] if kw else [LinearZeRO3(24, 8, None)])
    for m in mods:
        torch.nn.init.normal_(m.weight)
        kept = F.pack8(x, "int8")
        y = m(x, kept=kept)
        assert torch.equal(y, m(x))
        dx, dw = torch.autograd.grad(y, (x, m.weight), dy)
        assert torch.equal(dw, dy.t() @ kept.restore()) and torch.equal(dx, dy @ m.weight)
        with pytest.raises(ValueError):
            m(x, kept=F.pack8(x[:4]))


def test_separate_projections(monkeypatch):
    """q, k and v projections of their own read one kept row."""
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import ParallelContext
    from odysseus_transformer_b200.models.llama import LlamaForCausalLM
    _lossless(monkeypatch)
    cfg, ids = get_model_config("tiny-gqa", num_hidden_layers=1), torch.randint(32000, (1, 17), generator=_gen(1))
    grads = []
    for a8 in (None, "e4m3"):
        m = LlamaForCausalLM(cfg, "tpsp", ParallelContext(), pack_qkv=False, activations8=a8)
        m.init_weights(0)
        m(ids[:, :-1], torch.arange(16).unsqueeze(0), labels=ids[:, 1:]).backward()
        grads.append({k: p.grad for k, p in m.named_parameters()})
    for k, g in grads[0].items():
        torch.testing.assert_close(grads[1][k], g, rtol=1e-5, atol=1e-7)


def test_launches_are_counted_from_many_threads(tmp_path):
    """Backward passes count their launches from autograd's threads, without the interpreter's lock: none is lost."""
    import ctypes
    import os
    import subprocess
    from odysseus_transformer_b200.ops import native
    (tmp_path / "hammer.c").write_text("""
        #include <pthread.h>
        static void (*count)(long);
        static void* run(void* n) { for (long i = 0; i < (long)n; ++i) count(1); return 0; }
        void hammer(void (*f)(long), int threads, long n) {
          pthread_t t[16];
          count = f;
          for (int i = 0; i < threads; ++i) pthread_create(&t[i], 0, run, (void*)n);
          for (int i = 0; i < threads; ++i) pthread_join(t[i], 0);
        }""")
    so = str(tmp_path / "hammer.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-pthread", "-o", so, str(tmp_path / "hammer.c")], check=True)
    lib = native.lib()
    count = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(native.__file__)), "_C.so"))._Z18ody_count_launchesl
    lib.reset_launch_count()
    ctypes.CDLL(so).hammer(count, 4, ctypes.c_long(300000))
    assert lib.launch_count() == 4 * 300000
    lib.reset_launch_count()


def test_command_lines(capsys):
    import json
    from odysseus_transformer_b200.train import build_parser, main
    from odysseus_transformer_b200.utils import memory
    for extra in ([], ["--grad-checkpoint"]):
        out = main(build_parser().parse_args(["--model-config", "tiny", "--seq-length", "32", "--max-train-steps", "2", "--dtype", "fp32",
                                              "--parallel_mode", "odysseus", "--warmup-iterations", "0", "--activations8", "int8"] + extra))
        assert math.isfinite(out["loss"])
    capsys.readouterr()
    saved = []
    for extra in ([], ["--activations8"]):
        assert memory.main(["--model", "llama2-7b", "--seq-length", "16384", "--gpus", "1"] + extra) == 0
        saved.append(json.loads(capsys.readouterr().out)["saved_activations"])
    assert 0.45 < saved[1] / saved[0] < 0.55


def test_model_refuses_and_keeps_the_setting():
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import ParallelContext
    from odysseus_transformer_b200.models.llama import LlamaForCausalLM
    from odysseus_transformer_b200.parallel.apply import apply_seq_parallel
    from odysseus_transformer_b200.train import build_parser
    cfg, ctx = get_model_config("tiny", num_hidden_layers=1), ParallelContext()
    with pytest.raises(ValueError):
        LlamaForCausalLM(cfg, None, ctx, activations8="fp4")
    m = LlamaForCausalLM(cfg, None, ctx, activations8="int8")
    m.init_weights(0)
    assert apply_seq_parallel(m, "odysseus", ctx).layers[0].activations8 == "int8"
    assert build_parser().parse_args(["--activations8", "e4m3"]).activations8 == "e4m3"
    assert build_parser().parse_args([]).activations8 is None
    with torch.no_grad():                               # evaluation keeps nothing
        ids = torch.arange(8).unsqueeze(0)
        assert torch.equal(m(ids, ids), LlamaForCausalLM.forward(m, ids, ids))


@pytest.mark.parametrize("checkpoint", [False, True])
def test_models_pickled_without_the_setting(checkpoint):
    """A model that was saved whole before there was the setting runs as it did."""
    import io
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import ParallelContext
    from odysseus_transformer_b200.models.llama import LlamaForCausalLM
    m = LlamaForCausalLM(get_model_config("tiny", num_hidden_layers=1), "odysseus", ParallelContext())
    m.init_weights(0)
    if checkpoint:
        m.gradient_checkpointing_enable()
    ids = torch.arange(8).unsqueeze(0)
    want = m(ids, ids, labels=ids)
    for part in (m, *m.layers):
        part.__dict__.pop("activations8", None)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    loss = torch.load(f, weights_only=False)(ids, ids, labels=ids)
    assert torch.equal(loss, want)
    loss.backward()


@pytest.mark.parametrize("mode", ["odysseus", "ulysses", None])
def test_memory_estimate_of_kept_activations(mode):
    """The estimate's term against the bytes that autograd saves."""
    from odysseus_transformer_b200.config import get_model_config
    from odysseus_transformer_b200.mesh import ParallelContext
    from odysseus_transformer_b200.models.llama import LlamaForCausalLM
    from odysseus_transformer_b200.utils.memory import estimate_memory, saved_bytes_per_token_per_layer
    cfg, L = get_model_config("tiny"), 128
    m = LlamaForCausalLM(cfg, mode, ParallelContext(), activations8="e4m3")
    m.init_weights(0)
    seen = {}
    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: (seen.setdefault(t.untyped_storage().data_ptr(), (t.untyped_storage().nbytes(), t)), t)[1], lambda t: t):
        ids = torch.randint(cfg.vocab_size, (1, L))
        loss = m(ids, torch.arange(L).unsqueeze(0), labels=ids)
    params = {p.untyped_storage().data_ptr() for p in m.parameters()}
    kept = sum(nb for k, (nb, t) in seen.items() if k not in params and t.shape[-1] != cfg.vocab_size and nb >= L * 8 and t.dtype != torch.int64)
    kept -= 2 * L * cfg.hidden_size * 4 + 2 * L * cfg.head_dim // 2 * 4         # the final norm's, the rotation's tables
    assert kept / (L * cfg.num_hidden_layers) == pytest.approx(saved_bytes_per_token_per_layer(cfg, mode, 1, False, 4, True), rel=0.03)
    del loss
    big = get_model_config("llama2-7b")
    a, b = (estimate_memory(big, "odysseus", 32768, 1, grad_checkpoint=c) for c in (False, True))
    a8, b8 = (estimate_memory(big, "odysseus", 32768, 1, grad_checkpoint=c, activations8=True) for c in (False, True))
    assert 0.45 < a8["saved_activations"] / a["saved_activations"] < 0.55
    assert math.isclose((b["peak_allocated"] - b8["peak_allocated"]) * 2 ** 30, 32 * 32768 * (2 * 4096 - 4096 - 128), rel_tol=1e-9)
