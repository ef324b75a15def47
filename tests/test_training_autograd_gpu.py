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
