"""The norms around a block and their gradients against the definition in 64 bits (B200 only).

Tolerances: half a step of bf16 (2^-8) of each rounded result; fp32 arithmetic of at most 64 roundings of 2^-24 of the
magnitudes that enter it (sums are trees of 8 + 5 + 5 additions at most); a column sum over n rows at most
(n + 128) 2^-24 of the sum of its terms' magnitudes, in any order."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF, ACC = 2.0**-8, 2.0**-18
KINDS = ["layer_norm", "rms_norm", "none"]
EPS = 1e-6


def _make(dev, lead, h, seed, per=("gate", "mul", "add"), dtype=torch.float32, branch=True):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)
    b = lead[0] if len(lead) == 2 else 1
    vec = lambda n, base: (base + 0.3 * mk(*((b, 1, h) if n in per else (h,)))).to(dtype).to(dev)
    x = (0.5 + mk(*lead, h)).to(torch.bfloat16).to(dev) if branch else None
    return {"x": x, "residual": (2 * mk(*lead, h) - 0.3).to(torch.bfloat16).to(dev), "gate": vec("gate", 0.4) if branch else None,
            "mul": vec("mul", 1.0), "add": vec("add", 0.0), "post_weight": (1 + 0.3 * mk(h)).to(dtype).to(dev) if branch else None,
            "grad_r": (0.1 * mk(*lead, h)).to(torch.bfloat16).to(dev), "grad_out": (0.1 * mk(*lead, h)).to(torch.bfloat16).to(dev)}


def _normal(t, kind):
    if kind == "none":
        return t
    m = t.mean(-1, keepdim=True) if kind == "layer_norm" else 0.0
    return (t - m) / ((t - m).square().mean(-1, keepdim=True) + EPS).sqrt()


def _forward(st, post, norm, residual=None):
    d = {n: None if t is None else t.double() for n, t in st.items()}
    one = torch.ones((), dtype=torch.float64, device=st["residual"].device)
    gate = one if d["gate"] is None else d["gate"]
    w = one if d["post_weight"] is None else d["post_weight"]
    r = d["residual"] + gate * (w * _normal(d["x"], post)) if d["x"] is not None else d["residual"]
    n = _normal(r, norm)
    mul = one if d["mul"] is None else d["mul"]
    add = one * 0 if d["add"] is None else d["add"]
    return r, n * mul + add, (n * mul).abs() + add.abs()


def _kw(st, post, norm):
    return dict(eps=EPS, post_norm=post, post_weight=st["post_weight"], norm_type=norm)


def _check_forward(pkg, st, post, norm):
    r, out = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **_kw(st, post, norm))
    rr, ro, mag = _forward(st, post, norm)
    assert r.dtype == out.dtype == torch.bfloat16
    scale = rr.abs() + rr.square().mean(-1, keepdim=True).sqrt()
    assert ((r.double() - rr).abs() <= HALF * rr.abs() + ACC * scale).all()
    # the statistics see r's fp32 error through 1 / deviation
    rel = 1.0 if norm == "none" else scale / (rr.var(-1, keepdim=True, unbiased=False) + EPS).sqrt()
    m = 1.0 if st["mul"] is None else st["mul"].double().abs()
    assert ((out.double() - ro).abs() <= HALF * ro.abs() + ACC * (mag + rel * m * (1 + scale * (norm == "none")))).all()
    return r


def _hat(x, kind):
    rstd = 1.0
    if kind != "none":
        c = x - x.mean(-1, keepdim=True) if kind == "layer_norm" else x
        rstd = 1 / (c.square().mean(-1, keepdim=True) + EPS).sqrt()
        x = c * rstd
    return x, rstd


def _hat_grad(g, hat, rstd, kind):
    """(gradient, magnitudes that enter it)."""
    if kind == "none":
        return g, g.abs()
    m0, m1 = g.mean(-1, keepdim=True) if kind == "layer_norm" else 0.0, (g * hat).mean(-1, keepdim=True)
    mag = g.abs() + g.abs().mean(-1, keepdim=True) + hat.abs() * (g * hat).abs().mean(-1, keepdim=True)
    return rstd * (g - m0 - hat * m1), rstd * mag


def _backward(st, r, post, norm):
    """{name: (gradient, bound)} in fp64, from the stored r."""
    d = {n: None if t is None else t.double() for n, t in st.items()}
    one = torch.ones((), dtype=torch.float64, device=r.device)
    mul = one if d["mul"] is None else d["mul"]
    n, rstd = _hat(r.double(), norm)
    go = d["grad_out"] if d["grad_out"] is not None else torch.zeros_like(n)
    g, gmag = _hat_grad(go * mul, n, rstd, norm)
    gr = d["grad_r"] if d["grad_r"] is not None else torch.zeros_like(n)
    dr, rmag = gr + g, gr.abs() + gmag
    rows = r.numel() // r.shape[-1]

    def total(t, name):
        v = st[name]
        return t.reshape(v.shape[0], -1, v.shape[-1]).sum(1, keepdim=True) if v.dim() == 3 else t.flatten(0, -2).sum(0).reshape(v.shape)

    def col(t, mag, name):
        return total(t, name), (rows + 128) * 2.0**-24 * total(mag, name) + torch.finfo(st[name].dtype).eps / 2 * total(t, name).abs()

    res = {"residual": (dr, HALF * dr.abs() + ACC * rmag)}
    cond = 1.0 if norm == "none" else (r.double().abs().mean(-1, keepdim=True) * rstd)  # of the centring
    if d["mul"] is not None:
        res["mul"] = col(go * n, go.abs() * (n.abs() + cond), "mul")
    if d["add"] is not None:
        res["add"] = col(go, go.abs(), "add")
    if d["x"] is not None:
        y, rx = _hat(d["x"], post)
        gate = one if d["gate"] is None else d["gate"]
        w = one if d["post_weight"] is None else d["post_weight"]
        dx, xmag = _hat_grad(dr * gate * w, y, rx, post)
        _, emag = _hat_grad(rmag * (gate * w).abs(), y, rx, post)
        res["x"] = (dx, HALF * dx.abs() + ACC * (xmag + emag))
        ycond = 0.0 if post == "none" else d["x"].abs().mean(-1, keepdim=True) * rx
        if d["gate"] is not None:
            res["gate"] = col(dr * y * w, rmag * (y.abs() + ycond) * w.abs(), "gate")
        if d["post_weight"] is not None:
            res["post_weight"] = col(dr * y * gate, rmag * (y.abs() + ycond) * gate.abs(), "post_weight")
    return res


def _check_backward(pkg, st, r, post, norm):
    got = pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], r, st["gate"], st["mul"], st["add"], **_kw(st, post, norm))
    want = _backward(st, r, post, norm)
    for name in ("x", "residual", "gate", "mul", "add", "post_weight"):
        g = getattr(got, name)
        if name not in want:
            assert g is None, name
            continue
        ref, bound = want[name]
        assert g.shape == st[name].shape and g.dtype == st[name].dtype, name
        over = ((g.double() - ref).abs() / (bound + 1e-30)).max().item()
        assert over <= 1.0, f"{name}: {over:.3f} of the bound"
    return got


@pytest.mark.parametrize("post,norm", list(itertools.product(KINDS, KINDS)))
def test_kinds(pkg, dev, post, norm):
    st = _make(dev, (2, 37), 520, 1)
    _check_backward(pkg, st, _check_forward(pkg, st, post, norm), post, norm)


@pytest.mark.parametrize("lead,h", [((1,), 8), ((3,), 64), ((1, 1), 256), ((2, 5), 264), ((700,), 1536), ((1, 333), 5120),
                                    ((3, 3), 8192), ((1, 40), 8184), ((5, 1), 128), ((1, 2000), 72)])
def test_sizes(pkg, dev, lead, h):
    st = _make(dev, lead, h, h)
    _check_backward(pkg, st, _check_forward(pkg, st, "rms_norm", "layer_norm"), "rms_norm", "layer_norm")


@pytest.mark.parametrize("per", [(), ("gate",), ("mul", "add"), ("add",)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_and_per_batch_vectors(pkg, dev, per, dtype):
    st = _make(dev, (3, 21), 384, 2, per, dtype)
    _check_backward(pkg, st, _check_forward(pkg, st, "layer_norm", "rms_norm"), "layer_norm", "rms_norm")


@pytest.mark.parametrize("absent", [("gate",), ("mul", "add"), ("post_weight",), ("gate", "mul", "add", "post_weight")])
def test_absent_vectors(pkg, dev, absent):
    st = _make(dev, (2, 11), 640, 3)
    for n in absent:
        st[n] = None
    _check_backward(pkg, st, _check_forward(pkg, st, "rms_norm", "layer_norm"), "rms_norm", "layer_norm")


def test_without_branch(pkg, dev):
    """x=None: the differentiable form of adaln_modulate's first norm."""
    st = _make(dev, (2, 50), 1024, 4, branch=False)
    r, out = pkg.sandwich_norm(None, st["residual"], mul=st["mul"], add=st["add"], eps=EPS)
    assert r is st["residual"]
    _check_backward(pkg, st, r, "rms_norm", "layer_norm")
    ref = pkg.adaln_modulate(st["residual"], st["mul"], st["add"], eps=EPS, norm_type="layer_norm").double()
    # adaln_modulate rounds mul and add to bf16 first: one more half step of each
    mag = (out.double() - st["add"].double()).abs() + st["add"].double().abs()
    assert ((out.double() - ref).abs() <= 2 * HALF * ref.abs() + 1.01 * HALF * mag + ACC * 8).all()


@pytest.mark.parametrize("missing", ["grad_r", "grad_out"])
def test_one_gradient(pkg, dev, missing):
    st = _make(dev, (2, 9), 264, 5)
    r = _check_forward(pkg, st, "rms_norm", "layer_norm")
    st[missing] = None
    got = _check_backward(pkg, st, r, "rms_norm", "layer_norm")
    if missing == "grad_out":
        assert not got.mul.any() and not got.add.any()


def test_constant_and_zero_rows(pkg, dev):
    """Rows without variance: eps carries the norm, nothing is infinite."""
    st = _make(dev, (1, 4), 256, 6)
    st["x"][:, 1] = 0
    st["x"][:, 2] = 3.0
    st["residual"][:, 1] = 0
    st["residual"][:, 3] = -2.0
    for post, norm in itertools.product(KINDS, KINDS):
        r, out = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **_kw(st, post, norm))
        got = pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], r, st["gate"], st["mul"], st["add"], **_kw(st, post, norm))
        assert all(torch.isfinite(t).all() for t in (r, out, *got))


def test_views_and_empty(pkg, dev):
    st = _make(dev, (2, 20), 128, 7)
    want = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **_kw(st, "rms_norm", "layer_norm"))
    wide = torch.cat([st["x"], st["x"]], dim=-1)[..., 128:]
    turned = st["residual"].transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(st["gate"].numel() + 1, device=dev)[1:].view(st["gate"].shape).copy_(st["gate"])
    got = pkg.sandwich_norm(wide, turned, odd, st["mul"], st["add"], **_kw(st, "rms_norm", "layer_norm"))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    e = torch.empty(2, 0, 128, dtype=torch.bfloat16, device=dev)
    r, out = pkg.sandwich_norm(e, e, st["gate"], st["mul"], st["add"], eps=EPS)
    assert r.shape == out.shape == e.shape
    g = pkg.sandwich_norm_bwd(e, e, e, e, st["gate"], st["mul"], st["add"], eps=EPS)
    assert g.x.shape == e.shape and not g.gate.any() and not g.add.any()


def test_differentiable_form(pkg, dev):
    st = _make(dev, (2, 33), 512, 8)
    names = ("x", "residual", "gate", "mul", "add", "post_weight")
    for n in names:
        st[n].requires_grad_(True)
    r, out = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **_kw(st, "rms_norm", "layer_norm"))
    grads = torch.autograd.grad((r, out), [st[n] for n in names], (st["grad_r"], st["grad_out"]))
    for t in st.values():
        t.requires_grad_(False)
    want = pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], r.detach(), st["gate"], st["mul"], st["add"],
                                 **_kw(st, "rms_norm", "layer_norm"))
    for n, g in zip(names, grads):
        assert torch.equal(g, getattr(want, n)), n
    # broadcast and partly needed inputs
    gate = st["gate"][:1].clone().requires_grad_(True)
    _, out = pkg.sandwich_norm(st["x"], st["residual"], gate.expand(2, 1, 512), eps=EPS)
    (dg,) = torch.autograd.grad(out, gate, st["grad_out"])
    assert dg.shape == (1, 1, 512)
    full = pkg.sandwich_norm_bwd(None, st["grad_out"], st["x"], pkg.sandwich_norm(st["x"], st["residual"], gate.expand(2, 1, 512), eps=EPS)[0].detach(),
                                 gate.detach().expand(2, 1, 512), eps=EPS)
    assert torch.allclose(dg, full.gate.sum(0, keepdim=True), rtol=0, atol=1e-6 * full.gate.abs().max().item())


def test_against_differences(pkg, dev):
    """Directional derivatives by central differences of the 64-bit forward (the residual rounded as it was stored)."""
    st = _make(dev, (2, 6), 64, 9)
    post, norm = "rms_norm", "layer_norm"
    r = _check_forward(pkg, st, post, norm)
    got = _check_backward(pkg, st, r, post, norm)
    bounds = _backward(st, r, post, norm)
    st64 = {n: t.double() for n, t in st.items()}
    rr, _, _ = _forward(st64, post, norm)
    off = r.double() - rr  # the stored residual's rounding, held fixed
    h = 1e-6

    def loss(s):
        a = _forward(s, post, norm)[0] + off
        n = _normal(a, norm)
        return (a * st64["grad_r"]).sum() + ((n * s["mul"] + s["add"]) * st64["grad_out"]).sum()

    for name in ("x", "residual", "gate", "mul", "add", "post_weight"):
        u = torch.randn(st[name].shape, generator=torch.Generator().manual_seed(10), dtype=torch.float64).to(dev)
        slope = (loss({**st64, name: st64[name] + h * u}) - loss({**st64, name: st64[name] - h * u})) / (2 * h)
        room = (bounds[name][1] * u.abs()).sum() + 1e-6
        assert (getattr(got, name).double().mul(u).sum() - slope).abs() <= room, name


def test_same_bits_streams_capture(pkg, dev):
    st = _make(dev, (2, 700), 1536, 11)
    call = lambda r: pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], r, st["gate"], st["mul"], st["add"],
                                           **_kw(st, "rms_norm", "layer_norm"))
    r, _ = pkg.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **_kw(st, "rms_norm", "layer_norm"))
    first = call(r)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = [call(r) for _ in range(3)]
    here = [call(r) for _ in range(3)]
    torch.cuda.synchronize()
    for g in other + here:
        assert all(torch.equal(a, b) for a, b in zip(first, g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(r)
    st["grad_out"].mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    again = call(r)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
