"""Rotary positions with several axes against complex rotation in 64 bits (B200 only).

Tolerance: half a step of the output type, relative, plus 2^-20 of |x1| + |x2| for the fp32 arithmetic (the reduced
angle rounded to fp32, at most pi 2^-24; cosine and sine within 2 steps of 2^-24; two products and a sum)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _reference(x, pos, axes, theta, half, inverse):
    """(rotated x, |x1| + |x2|) in fp64."""
    d = x.shape[-1]
    y, mag = torch.empty(x.shape, dtype=torch.float64, device=x.device), torch.empty(x.shape, dtype=torch.float64, device=x.device)
    pair = 0
    for a, n in enumerate(axes):
        for i in range(n // 2):
            i1, i2 = (pair, pair + d // 2) if half else (2 * pair, 2 * pair + 1)
            ang = (pos[..., a].double() * theta ** (-2 * i / n))[..., None] * (-1 if inverse else 1)
            x1, x2 = x[..., i1].double(), x[..., i2].double()
            y[..., i1], y[..., i2] = x1 * ang.cos() - x2 * ang.sin(), x2 * ang.cos() + x1 * ang.sin()
            mag[..., i1] = mag[..., i2] = x1.abs() + x2.abs()
            pair += 1
    return y, mag


def _check(got, x, pos, axes, theta=10000.0, half=False, inverse=False):
    ref, mag = _reference(x, pos, axes, theta, half, inverse)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    bound = torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0**-20 * mag
    if x.dtype == torch.float16:
        bound = bound + 2.0**-25  # half a step of a subnormal
    assert ((got.double() - ref).abs() <= bound).all()


def _qk(dev, b, s, hq, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(b, s, h, d, generator=g).to(dtype).to(dev) for h in (hq, hk)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("b,s,hq,hk,axes", [(1, 1, 1, 1, (44, 42, 42)), (2, 77, 6, 2, (16, 56, 56)), (1, 130, 40, 40, (44, 42, 42)),
                                            (1, 33, 3, 3, (64,)), (2, 9, 5, 1, (8, 4, 2, 2)), (1, 600, 2, 2, (128, 128)),
                                            (1, 5, 7, 7, (24, 24))])
def test_against_definition(pkg, dev, dtype, pairing, b, s, hq, hk, axes):
    q, k = _qk(dev, b, s, hq, hk, sum(axes), dtype, s)
    pos = torch.randint(-50, 5000, (b, s, len(axes)), generator=torch.Generator().manual_seed(1)).to(dev)
    for inverse in (False, True):
        a, c = pkg.rotary_axes(q, k, pos, axes, pairing=pairing, inverse=inverse)
        _check(a, q, pos, axes, half=pairing == "half", inverse=inverse)
        _check(c, k, pos, axes, half=pairing == "half", inverse=inverse)
        assert torch.equal(pkg.rotary_axes(q, None, pos, axes, pairing=pairing, inverse=inverse), a)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64, torch.float32])
def test_positions(pkg, dev, pos_dtype):
    """Far, negative and fractional positions; one table for the batch or one per element."""
    q, k = _qk(dev, 2, 40, 3, 3, 128, torch.float32)
    far = torch.randint(-(1 << 23), 1 << 23, (2, 40, 3), generator=torch.Generator().manual_seed(2)).to(dev)
    pos = far.to(pos_dtype) if pos_dtype != torch.float32 else far.float() / 7
    a, c = pkg.rotary_axes(q, k, pos, (44, 42, 42), theta=256.0)
    _check(a, q, pos, (44, 42, 42), theta=256.0)
    _check(c, k, pos, (44, 42, 42), theta=256.0)
    shared = pos[:1].expand(2, -1, -1)
    x = pkg.rotary_axes(q, k, pos[0], (44, 42, 42))
    y = pkg.rotary_axes(q, k, shared, (44, 42, 42))
    assert all(torch.equal(m, n) for m, n in zip(x, y))


def test_wan_tables(pkg, dev):
    """The framework's own host tables and interleaved rotation, on a clip's patches."""
    from importlib import import_module

    rope = import_module("vllm-omni-neuron_b200.rope")
    latent = (5, 8, 14)
    cos, sin = rope.wan_rotary_freqs(128, (1, 2, 2), 1024, latent, device=dev)
    pos = pkg.wan_grid_positions(latent, (1, 2, 2), dev)
    assert pos.shape == (5 * 4 * 7, 3) and pos.dtype == torch.int32
    q, k = _qk(dev, 1, pos.shape[0], 4, 4, 128, torch.float32)
    a, c = pkg.rotary_axes(q, k, pos, (44, 42, 42))
    for x, y in ((a, q), (c, k)):
        assert ((x - rope.apply_rotary_emb_wan(y, cos, sin)).abs() <= 2.0**-20 * y.abs().amax()).all()


def test_views(pkg, dev):
    b, s, hq, hk, d = 2, 50, 4, 2, 128
    fused = torch.randn(b, s, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    q, k, _ = (t.unflatten(2, (-1, d)) for t in fused.split([hq * d, hk * d, hk * d], dim=2))
    pos = pkg.wan_grid_positions((50, 1, 1), (1, 1, 1), dev)
    axes = (44, 42, 42)
    want = pkg.rotary_axes(q.contiguous(), k.contiguous(), pos, axes)
    head_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=dev)[1:].view(k.shape).copy_(k)
    wide = torch.zeros(b, s, hq, 2 * d, dtype=q.dtype, device=dev)
    wide[..., ::2] = q
    for x, y in ((q, k), (head_major, odd), (wide[..., ::2], k)):
        assert all(torch.equal(m, n) for m, n in zip(want, pkg.rotary_axes(x, y, pos, axes)))
    one = k[:, :, :1].expand(b, s, hk, d)
    assert torch.equal(pkg.rotary_axes(q, one, pos, axes)[1], pkg.rotary_axes(q, one.contiguous(), pos, axes)[1])
    row = q[:, :1].expand(b, s, hq, d)  # one token, broadcast
    assert torch.equal(pkg.rotary_axes(row, k, pos, axes)[0], pkg.rotary_axes(row.contiguous(), k, pos, axes)[0])
    assert torch.equal(pkg.rotary_axes(q, k, pos.expand(2, -1, -1), axes)[0], want[0])


def test_empty(pkg, dev):
    e = torch.empty(1, 0, 4, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.empty(0, 3, dtype=torch.int32, device=dev)
    a, c = pkg.rotary_axes(e, e, pos, (44, 42, 42))
    assert a.shape == e.shape and c.shape == e.shape


@pytest.mark.parametrize("only", ["q", "k", "both"])
def test_gradient(pkg, dev, only):
    """The gradient is the inverse rotation: <R x, g> = <x, R^T g>, by formula and as a difference (R is linear)."""
    q, k = _qk(dev, 1, 21, 3, 1, 64, torch.float32)
    pos, axes = torch.rand(1, 21, 2, generator=torch.Generator().manual_seed(4)).to(dev) * 30, (24, 40)
    q.requires_grad_(only != "k")
    k.requires_grad_(only != "q")
    a, c = pkg.rotary_axes(q, k, pos, axes)
    gq, gk = torch.randn_like(a), torch.randn_like(c)
    leaves = [t for t in (q, k) if t.requires_grad]
    loss = (a * gq).sum() * (only != "k") + (c * gk).sum() * (only != "q")
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(loss, leaves)))
    for t, g, out in ((q, gq, a), (k, gk, c)):
        if not t.requires_grad:
            continue
        got = grads[id(t)]
        _check(got, g, pos, axes, inverse=True)
        u = torch.randn_like(t)
        moved = pkg.rotary_axes((t + u).detach(), None, pos, axes)
        slope = ((moved.double() - out.detach().double()) * g.double()).sum()
        # fp32 rounding of the two ends, 2^-20 of the magnitudes each
        room = 2.0**-19 * ((t.abs() + u.abs()).sum(-1, keepdim=True).double() * g.double().abs()).sum()
        assert (got.double().mul(u.double()).sum() - slope).abs() <= room


def test_streams_and_capture(pkg, dev):
    q, k = _qk(dev, 1, 64, 4, 4, 128, torch.bfloat16)
    pos, axes = pkg.wan_grid_positions((64, 1, 1), (1, 1, 1), dev), (44, 42, 42)
    want = pkg.rotary_axes(q, k, pos, axes)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = pkg.rotary_axes(q, k, pos, axes)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.rotary_axes(q, k, pos, axes)
    q.copy_(k.flip(1))
    pos.add_(5)
    graph.replay()
    torch.cuda.synchronize()
    _check(out[0], q, pos, axes)
