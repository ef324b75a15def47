"""Refusals of a gradient of the log-sum-exp, and its fake shapes (CPU)."""

import pytest
import torch


def test_refusals(pkg):
    q = torch.zeros(1, 130, 2, 128, dtype=torch.bfloat16)
    o, lse = torch.zeros(1, 2, 130, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 128, 2)
    with pytest.raises(ValueError, match="grad_lse"):
        pkg.attention_bwd(o, q, q, q, o, lse, grad_lse=torch.zeros(1, 2, 2, 128))
    with pytest.raises(ValueError, match="grad_lse"):
        pkg.attention_bwd(o, q, q, q, o, lse, grad_lse=lse.int())
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.attention_bwd(o, q, q, q, o, lse, grad_lse=lse)


def test_fake_gradient_through_lse(pkg):
    mk = lambda *s: torch.empty(*s, device="meta", dtype=torch.bfloat16).requires_grad_(True)
    q, k, v = mk(1, 64, 4, 128), mk(1, 70, 2, 128), mk(1, 70, 2, 128)
    o, lse = torch.ops.b200omni.attention_fwd(q, k, v)
    for loss in (lse.sum(), o.sum(), lse.sum() + o.float().sum()):
        assert [t.shape for t in torch.autograd.grad(loss, (q, k, v), retain_graph=True)] == [q.shape, k.shape, v.shape]
