"""What autograd sees of the training functions, on the CPU: tangents are refused before any device call."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_gradient_functions_refuse_tangents(pkg):
    q, o, lse, x = _bf(1, 16, 2, 128), _bf(1, 2, 16, 128), torch.zeros(1, 2, 128, 1), _bf(1, 8, 64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for i in range(6):
            args = [o, q, q, q, o, lse]
            args[i] = dual(args[i])
            with pytest.raises(NotImplementedError):
                pkg.attention_bwd(*args)
        with pytest.raises(NotImplementedError):
            pkg.attention_bwd(o, q, q, q, o, lse, grad_lse=dual(lse))
        for i in range(4):
            args = [x, x, x, x]
            args[i] = dual(x)
            with pytest.raises(NotImplementedError):
                pkg.sandwich_norm_bwd(*args, eps=1e-6)
        with pytest.raises(RuntimeError, match="CPU"):  # no tangent: on to the next check
            pkg.attention_bwd(o, q, q, q, o, lse)
