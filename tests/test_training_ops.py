"""The training operators as torch custom operators: registration and fake (meta) shapes, on the CPU."""

import torch

M = torch.device("meta")


def _e(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device=M, dtype=dtype)


def test_fake_shapes(pkg):
    ops = torch.ops.b200omni
    q, k = _e(2, 300, 40, 128), _e(2, 512, 8, 128)
    o, lse = ops.attention_fwd(q, k, k, None, None, [512, 3])
    assert o.shape == (2, 40, 300, 128) and lse.shape == (2, 40, 128, 3) and lse.dtype == torch.float32
    assert [t.shape for t in ops.attention_bwd(o, q, k, k, o, lse)] == [q.shape, k.shape, k.shape]
    pos = _e(300, 3, dtype=torch.int32)
    assert [t.shape for t in ops.rotary_axes(q, _e(2, 300, 8, 128), pos, [44, 42, 42])] == [q.shape, (2, 300, 8, 128)]
    assert len(ops.rotary_axes(q, None, pos, [44, 42, 42], 10000.0, "half", True)) == 1
    x, g, w = _e(2, 300, 5120), _e(2, 1, 5120, dtype=torch.float32), _e(5120, dtype=torch.float32)
    assert [t.shape for t in ops.sandwich_norm(x, x, g, g, None, 1e-6)] == [x.shape, x.shape]
    assert len(ops.sandwich_norm(None, x, None, g, g, 1e-6)) == 1
    grads = ops.sandwich_norm_bwd(x, x, x, x, g, g, None, 1e-6, "rms_norm", w)
    assert [t.shape for t in grads] == [x.shape, x.shape, g.shape, g.shape, w.shape] and grads[2].dtype == torch.float32


def test_fake_gradients(pkg):
    """The registered derivatives give every input a gradient of its shape."""
    ops = torch.ops.b200omni
    q, k = (t.requires_grad_(True) for t in (_e(1, 64, 4, 128), _e(1, 64, 2, 128)))
    a, c = ops.rotary_axes(q, k, _e(64, 3, dtype=torch.int32), [44, 42, 42])
    o, _ = ops.attention_fwd(a, c, c)
    assert [t.shape for t in torch.autograd.grad(o.sum(), (q, k))] == [q.shape, k.shape]
    x, w = _e(1, 64, 512).requires_grad_(True), _e(512, dtype=torch.float32).requires_grad_(True)
    r, out = ops.sandwich_norm(x, _e(1, 64, 512), None, w, None, 1e-6, "rms_norm", w)
    assert [t.shape for t in torch.autograd.grad(out.sum(), (x, w))] == [x.shape, w.shape]
