"""The training operators together, as a trainable self-attention sub-layer: norm, projection, rotary positions, attention,
projection, gated residual with norms before and after (B200 only)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

AXES = (44, 42, 42)


def _weights(dev, b, h, heads, kv_heads):
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g)
    w = {"qkv": mk(h, (heads + 2 * kv_heads) * 128) / math.sqrt(h), "o": mk(heads * 128, h) / math.sqrt(heads * 128)}
    w = {n: t.to(torch.bfloat16).to(dev) for n, t in w.items()}
    vec = {"mul": 1 + 0.1 * mk(b, 1, h), "add": 0.1 * mk(b, 1, h), "gate": 0.7 + 0.1 * mk(b, 1, h), "post": 1 + 0.1 * mk(h),
           "mul2": 1 + 0.1 * mk(h), "add2": 0.1 * mk(h)}
    return {**w, **{n: t.to(dev) for n, t in vec.items()}}


def _sublayer(pkg, x, w, pos, heads, kv_heads, lens):
    _, n1 = pkg.sandwich_norm(None, x, mul=w["mul"], add=w["add"], eps=1e-6)
    qkv = n1 @ w["qkv"]
    q, k, v = (t.unflatten(2, (-1, 128)) for t in qkv.split([heads * 128, kv_heads * 128, kv_heads * 128], dim=2))
    q, k = pkg.rotary_axes(q, k, pos, AXES)
    o = pkg.wan_attention(q, k, v, q_lens=lens, kv_lens=lens)
    return pkg.sandwich_norm(o.transpose(1, 2).flatten(2) @ w["o"], x, w["gate"], w["mul2"], w["add2"], eps=1e-6,
                             post_weight=w["post"])


def _plain(x, w, pos, heads, kv_heads, lens):
    """The same in 64 bits with plain operations."""
    def ln(t):
        return (t - t.mean(-1, keepdim=True)) / (t.var(-1, keepdim=True, unbiased=False) + 1e-6).sqrt()

    freqs = torch.cat([10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64, device=x.device) / n) for n in AXES])
    axis = torch.repeat_interleave(torch.arange(3, device=x.device), torch.tensor([n // 2 for n in AXES], device=x.device))
    ang = (pos.double()[..., axis] * freqs).unsqueeze(-2)

    def turn(t):
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).flatten(-2)

    qkv = (ln(x) * w["mul"] + w["add"]) @ w["qkv"]
    q, k, v = (t.unflatten(2, (-1, 128)) for t in qkv.split([heads * 128, kv_heads * 128, kv_heads * 128], dim=2))
    q, k = turn(q).transpose(1, 2), turn(k).transpose(1, 2)
    k, v = (t.repeat_interleave(heads // kv_heads, dim=1) for t in (k, v.transpose(1, 2)))
    s = q @ k.transpose(2, 3) / math.sqrt(128)
    if lens:
        keep = torch.arange(s.shape[-1], device=x.device)[None] < torch.tensor(lens, device=x.device)[:, None]
        p = torch.softmax(s.masked_fill(~keep[:, None, None, :], -1e300), -1) * keep[:, None, :, None] * keep[:, None, None, :]
    else:
        p = torch.softmax(s, -1)
    a = (p @ v).transpose(1, 2).flatten(2) @ w["o"]
    y = a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w["post"]
    r = x + w["gate"] * y
    return r, ln(r) * w["mul2"] + w["add2"]


@pytest.mark.parametrize("heads,kv_heads,lens", [(4, 4, None), (6, 2, None), (4, 2, [260, 131])])
def test_gradients(pkg, dev, heads, kv_heads, lens):
    """Every gradient is within 16 half steps of bf16 of the 64-bit one, in norm: eight results are rounded to bf16 on the way
    forward (norm, qkv, rotary, P, o, projection, residual, norm) and eight on the way back, and no stage enlarges a
    relative error of a typical direction."""
    b, s, h = 2, 260, 512
    w = _weights(dev, b, h, heads, kv_heads)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(b, s, h, generator=g).to(torch.bfloat16).to(dev)
    grads = [torch.randn(b, s, h, generator=g).to(torch.bfloat16).to(dev) / 8 for _ in range(2)]
    if lens:  # padded tokens: no gradient comes from them
        for i, n in enumerate(lens):
            for t in grads:
                t[i, n:] = 0
    pos = pkg.wan_grid_positions((4, 5, 13), (1, 1, 1), dev)
    leaves = {"x": x, **w}
    for t in leaves.values():
        t.requires_grad_(True)
    got = torch.autograd.grad(_sublayer(pkg, x, w, pos, heads, kv_heads, lens), list(leaves.values()), grads)
    wide = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    want = torch.autograd.grad(_plain(wide["x"], {n: wide[n] for n in w}, pos, heads, kv_heads, lens), list(wide.values()),
                               [t.double() for t in grads])
    for name, a, c in zip(leaves, got, want):
        assert a.shape == c.shape and torch.isfinite(a).all(), name
        assert (a.double() - c).norm() <= 16 * 2.0**-8 * c.norm(), f"{name}: {(a.double() - c).norm() / c.norm():.4f}"


def test_the_framework_s_training_forward(pkg, dev):
    """ring_attention_const_max_fwd(training=True) gives what attention_bwd takes."""
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 300, 2, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(3))
    go = torch.randn(1, 2, 300, 128, generator=g).to(torch.bfloat16).to(dev)
    o, lse = pkg.ring_attention_const_max_fwd(q, k, v, training=True)
    o2, lse2 = pkg.attention_fwd(q, k, v)
    assert torch.equal(o, o2)
    rows = lse.transpose(2, 3).reshape(1, 2, -1)[:, :, :300]
    assert torch.equal(rows, lse2.transpose(2, 3).reshape(1, 2, -1)[:, :, :300])
    a, c = pkg.attention_bwd(go, q, k, v, o, lse), pkg.attention_bwd(go, q, k, v, o2, lse2)
    assert all(torch.equal(m, n) for m, n in zip(a, c))


def test_custom_operators(pkg, dev):
    """torch.ops.b200omni.* give the same results and gradients."""
    ops = torch.ops.b200omni
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    q, k, v, go = mk(1, 96, 4, 128), mk(1, 96, 2, 128), mk(1, 96, 2, 128), mk(1, 4, 96, 128)
    pos = pkg.wan_grid_positions((96, 1, 1), (1, 1, 1), dev)
    for t in (q, k, v):
        t.requires_grad_(True)
    a, c = pkg.rotary_axes(q, k, pos, AXES)
    want = torch.autograd.grad(pkg.wan_attention(a, c, v), (q, k, v), go)
    a, c = ops.rotary_axes(q, k, pos, list(AXES))
    got = torch.autograd.grad(ops.attention_fwd(a, c, v)[0], (q, k, v), go)
    assert all(torch.equal(m, n) for m, n in zip(want, got))
    x, r, gate, w = mk(1, 96, 512), mk(1, 96, 512), mk(1, 1, 512), mk(512)
    for t in (x, r, gate, w):
        t.requires_grad_(True)
    gr = [mk(1, 96, 512), mk(1, 96, 512)]
    want = torch.autograd.grad(pkg.sandwich_norm(x, r, gate, eps=1e-6, post_weight=w), (x, r, gate, w), gr)
    got = torch.autograd.grad(ops.sandwich_norm(x, r, gate, None, None, 1e-6, "rms_norm", w), (x, r, gate, w), gr)
    assert all(torch.equal(m, n) for m, n in zip(want, got))
    (got,) = torch.autograd.grad(ops.sandwich_norm(None, r, None, None, None, 1e-6)[0], r, gr[0])
    (want,) = torch.autograd.grad(pkg.sandwich_norm(None, r, eps=1e-6)[1], r, gr[0])
    assert torch.equal(got, want)


def test_a_step_captured_and_replayed(pkg, dev):
    """Forward and backward of the sub-layer in one graph, gradients asked for with autograd.grad."""
    b, s, h, heads = 1, 130, 256, 2
    w = _weights(dev, b, h, heads, heads)
    g = torch.Generator().manual_seed(4)
    mk = lambda: torch.randn(b, s, h, generator=g).to(torch.bfloat16).to(dev)
    x, gr = mk().requires_grad_(True), [mk(), mk()]
    pos = pkg.wan_grid_positions((130, 1, 1), (1, 1, 1), dev)
    leaves = [x] + [t.requires_grad_(True) for t in w.values()]
    step = lambda: torch.autograd.grad(_sublayer(pkg, x, w, pos, heads, heads, None), leaves, gr)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(mk())
        gr[0].copy_(mk())
    graph.replay()
    torch.cuda.synchronize()
    again = step()
    assert all(torch.equal(m, n) for m, n in zip(out, again))
