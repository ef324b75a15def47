"""Rows without variance (zeros, constants) through the norms around a block, against the definition in 64 bits (B200 only).

Tolerances. A mean is a sum in fp32, off by ACC = 64 * 2^-24 of the mean magnitude at most (trees of 8 + 5 + 5 additions), and so is every
value less its mean: in a constant row that is all there is, and 1 / sqrt(eps) = 1000 enlarges it. From there the errors are carried through
the formulas to the end, term by term, with fp32 roundings of ACC of the magnitudes that enter and half a step of bf16 (2^-8) of what is
rounded. A column sum over n rows is off by (n + 128) 2^-24 of its terms' magnitudes, in any order. At 512 columns the mean of a small whole
number is exact, so is its row of zeros, and out is add."""

import itertools

import pytest
import torch
from test_sandwich_gpu import ACC, EPS, HALF, KINDS, _make

pytestmark = pytest.mark.gpu


def _flat(st):
    """Every fifth row of x and of the stream: zeros, and two constants."""
    for name, at in (("x", ((1, 0.0), (2, 3.0), (3, -0.75))), ("residual", ((0, 0.0), (2, -2.0), (4, 5.5)))):
        if st[name] is not None:
            rows = st[name].view(-1, st[name].shape[-1])
            for i, value in at:
                rows[i::5] = value
    return st


def _hat(v, kind):
    """(hat, its error, 1 / deviation, its relative error) of the rows of v."""
    if kind == "none":
        return v, torch.zeros_like(v), torch.ones_like(v[..., :1]), torch.zeros_like(v[..., :1])
    c, e = v, 2.0**-24 * v.abs()
    if kind == "layer_norm":
        c, e = v - v.mean(-1, keepdim=True), e + ACC * v.abs().mean(-1, keepdim=True)
    q = c.square().mean(-1, keepdim=True)
    e_q = (2 * c.abs() * e + e * e).mean(-1, keepdim=True) + ACC * q
    rstd = 1 / (q + EPS).sqrt()
    rel = 0.75 * e_q / (q + EPS) + 2.0**-20
    return c * rstd, (e + c.abs() * rel) * rstd * (1 + rel), rstd, rel


def _hat_grad(g, e_g, hat, e_hat, rstd, rel, kind):
    """The gradient behind _hat and its error, of g with the error e_g."""
    if kind == "none":
        return g, e_g
    mean = lambda t: t.mean(-1, keepdim=True)
    m1 = mean(g * hat)
    e_m1 = ACC * mean((g * hat).abs()) + mean(e_g * hat.abs() + (g.abs() + e_g) * e_hat)
    m0, e_m0 = (mean(g), ACC * mean(g.abs()) + mean(e_g)) if kind == "layer_norm" else (0.0, 0.0)
    out = rstd * (g - m0 - hat * m1)
    return out, out.abs() * rel + rstd * (1 + rel) * (e_g + ACC * g.abs() + e_m0 + hat.abs() * e_m1 + e_hat * (m1.abs() + e_m1))


def _within(name, got, want, e):
    over = ((got.double() - want).abs() / (e + 1e-30)).max().item()
    assert torch.isfinite(got).all() and over <= 1.0, f"{name}: {over:.3f} of the bound"


LEADS = [((1, 4), 256), ((2, 5), 520), ((1, 3001), 520), ((1, 3001), 128), ((1, 1303), 5000), ((700,), 1536), ((1, 602), 6000)]


@pytest.mark.parametrize("lead,h", LEADS)
@pytest.mark.parametrize("post,norm", list(itertools.product(KINDS, KINDS)))
def test_backward(pkg, dev, lead, h, post, norm):
    st = _flat(_make(dev, lead, h, h))
    r = st["residual"]  # the stream as a forward pass may have stored it
    got = pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], r, st["gate"], st["mul"], st["add"], eps=EPS, post_norm=post,
                                post_weight=st["post_weight"], norm_type=norm)
    d = {n: t.double() for n, t in st.items()}
    n, e_n, rstd, rel = _hat(d["residual"], norm)
    go = d["grad_out"]
    g, e_g = _hat_grad(go * d["mul"], ACC * (go * d["mul"]).abs(), n, e_n, rstd, rel, norm)
    dr = d["grad_r"] + g
    e_dr = e_g + ACC * (d["grad_r"].abs() + g.abs())
    _within("residual", got.residual, dr, HALF * (dr.abs() + e_dr) + e_dr)
    y, e_y, rx, rel_x = _hat(d["x"], post)
    gw = d["gate"] * d["post_weight"]
    dx, e_dx = _hat_grad(dr * gw, (e_dr + ACC * dr.abs()) * gw.abs(), y, e_y, rx, rel_x, post)
    _within("x", got.x, dx, HALF * (dx.abs() + e_dx) + e_dx)
    rows = r.numel() // h

    def column(name, t, e, mag):
        v = st[name]
        total = lambda t: t.reshape(v.shape[0], -1, h).sum(1, keepdim=True) if v.dim() == 3 else t.flatten(0, -2).sum(0).reshape(v.shape)
        _within(name, getattr(got, name), total(t), total(e) + (rows + 128) * 2.0**-24 * total(mag + e))

    zero = torch.zeros_like(go)
    column("add", go + zero, zero, go.abs())
    column("mul", go * n, go.abs() * e_n, (go * n).abs())
    e_a, a = e_dr * (y.abs() + e_y) + dr.abs() * e_y, dr * y
    column("gate", a * d["post_weight"], e_a * d["post_weight"].abs() + ACC * (a * d["post_weight"]).abs(), (a * d["post_weight"]).abs())
    column("post_weight", a * d["gate"], e_a * d["gate"].abs() + ACC * (a * d["gate"]).abs(), (a * d["gate"]).abs())


@pytest.mark.parametrize("lead,h", LEADS)
@pytest.mark.parametrize("norm", KINDS)
def test_forward(pkg, dev, lead, h, norm):
    """The first norm of a block, and a gated residual without a post norm (whose stream is off by roundings alone)."""
    st = _flat(_make(dev, lead, h, h + 1))
    _, out = pkg.sandwich_norm(None, st["residual"], mul=st["mul"], add=st["add"], eps=EPS, norm_type=norm)
    d = {n: t.double() for n, t in st.items()}
    n, e_n, _, _ = _hat(d["residual"], norm)
    want = n * d["mul"] + d["add"]
    e = e_n * d["mul"].abs() + ACC * ((n * d["mul"]).abs() + d["add"].abs())
    _within("out", out, want, HALF * (want.abs() + e) + e)
    st["gate"][:] = 0.5  # products of bf16 values that fp32 holds: flat rows of r where both are flat
    r, out = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], eps=EPS, post_norm="none", norm_type=norm)
    rr = d["residual"] + 0.5 * d["x"]
    _within("residual_out", r, rr, HALF * rr.abs() + 2.0**-23 * (d["residual"].abs() + d["x"].abs()))
    r32 = (st["residual"].float() + 0.5 * st["x"].float()).double()  # fp32's one rounding of it
    n, e_n, _, _ = _hat(r32, norm)
    want = n * d["mul"] + d["add"]
    e = e_n * d["mul"].abs() + ACC * ((n * d["mul"]).abs() + d["add"].abs())
    _within("out behind the residual", out, want, HALF * (want.abs() + e) + e)


@pytest.mark.parametrize("rows", [3, 2000])
def test_exact_means(pkg, dev, rows):
    st = _make(dev, (1, rows), 512, 9)
    st["residual"][:] = torch.tensor([-3.0, 0.0, 7.0])[torch.arange(rows) % 3][None, :, None].to(torch.bfloat16).to(dev)
    _, out = pkg.sandwich_norm(None, st["residual"], mul=st["mul"], add=st["add"], eps=EPS)
    assert torch.equal(out, st["add"].to(torch.bfloat16).expand_as(out))
    got = pkg.sandwich_norm_bwd(None, st["grad_out"], None, st["residual"], mul=st["mul"], add=st["add"], eps=EPS)
    assert not got.mul.any()
