"""What autograd sees of the training functions: gradients of every result, and no tangent lost (B200 only)."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def _make(dev, seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


def _qkv(dev):
    return [_make(dev, i, 2, s, h, 128).requires_grad_(True) for i, (s, h) in enumerate(((130, 4), (70, 2), (70, 2)))]


@pytest.mark.parametrize("use", ["both", "o", "lse"])
@pytest.mark.parametrize("lens", [None, [70, 1]])
def test_attention_fwd(pkg, dev, use, lens):
    """The function is differentiable as the operator of its name, to the bit."""
    q, k, v = _qkv(dev)
    go, gl = _make(dev, 5, 2, 4, 130, 128), _make(dev, 6, 2, 4, 128, 2).float()
    gl.view(2, 4, 128, 2)[:, :, 2:, 1] = 0  # behind the rows, where lse is -inf
    pick = lambda r: {"both": (r, (go, gl)), "o": (r[:1], (go,)), "lse": (r[1:], (gl,))}[use]
    got = torch.autograd.grad(*map(tuple, pick(pkg.attention_fwd(q, k, v, kv_lens=lens))[:1]), (q, k, v), pick((0, 0))[1])
    want = torch.autograd.grad(tuple(pick(torch.ops.b200omni.attention_fwd(q, k, v, None, None, lens))[0]), (q, k, v), pick((0, 0))[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0].any() and (use == "lse" or got[2].any())


def test_no_graph_where_none_is_asked_for(pkg, dev):
    q, k, v = _qkv(dev)
    with torch.no_grad():
        o, lse = pkg.attention_fwd(q, k, v)
    assert not o.requires_grad and not lse.requires_grad
    o2, lse2 = pkg.attention_fwd(q, k, v)
    assert o2.requires_grad and lse2.requires_grad and torch.equal(o, o2) and torch.equal(lse, lse2)
    assert not pkg.attention_fwd(*(t.detach() for t in (q, k, v)))[0].requires_grad
    only = torch.autograd.grad(pkg.attention_fwd(q.detach(), k, v.detach())[0].sum(), k)  # one input alone
    assert only[0].shape == k.shape


def _calls(pkg, dev):
    q, x, g = _make(dev, 1, 1, 64, 2, 128), _make(dev, 2, 1, 64, 512), _make(dev, 3, 1, 1, 512).float()
    pos = pkg.wan_grid_positions((64, 1, 1), (1, 1, 1), dev)
    ops, axes = torch.ops.b200omni, (44, 42, 42)
    with torch.no_grad():
        o, lse = pkg.attention_fwd(q, q, q)
    return [
        (lambda t: pkg.rotary_axes(t, None, pos, axes), q),
        (lambda t: pkg.rotary_axes(q, t, pos, axes)[1], q),
        (lambda t: pkg.sandwich_norm(None, t, eps=1e-6)[1], x),
        (lambda t: pkg.sandwich_norm(t, x, eps=1e-6)[1], x),
        (lambda t: pkg.sandwich_norm(x, x, t, eps=1e-6)[0], g),
        (lambda t: pkg.sandwich_norm(x, x, mul=t, eps=1e-6)[1], g),
        (lambda t: pkg.attention_fwd(t, q, q)[0], q),
        (lambda t: pkg.attention_fwd(q, t, q)[1], q),
        (lambda t: pkg.wan_attention(q, q, t), q),
        (lambda t: pkg.attention_bwd(t, q, q, q, o, lse)[0], o),
        (lambda t: pkg.sandwich_norm_bwd(t, None, x, x, eps=1e-6).x, x),
        (lambda t: ops.rotary_axes(t, None, pos, list(axes))[0], q),
        (lambda t: ops.sandwich_norm(t, x, None, None, None, 1e-6)[0], x),
        (lambda t: ops.attention_fwd(t, q, q)[0], q),
        (lambda t: ops.attention_bwd(t, q, q, q, o, lse)[0], o),
        (lambda t: ops.sandwich_norm_bwd(t, None, x, x, None, None, None, 1e-6)[0], x),
    ]


@pytest.mark.parametrize("which", range(16))
def test_tangents_are_refused(pkg, dev, which):
    fn, t = _calls(pkg, dev)[which]
    want = fn(t)
    with forward_ad.dual_level():
        assert torch.equal(fn(t), want)  # an open level alone changes nothing
        with pytest.raises(NotImplementedError):
            fn(forward_ad.make_dual(t, torch.ones_like(t)))
    assert torch.equal(fn(t), want)
