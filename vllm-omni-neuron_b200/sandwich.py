"""Norms before and after a block, fused with its gate and residual, forward and backward.

``adaln_modulate`` normalises after the gated residual only; transformers that also normalise the sub-layer's output
before it enters the stream (a "sandwich") need

    y = post(x) * post_weight;   r = residual + gate * y;   out = norm(r) * mul + add

in one pass, and training needs its gradients. Without ``x`` the branch is absent and ``out = norm(residual) * mul + add``:
the differentiable form of the block's first norm. Vector layouts are those of ``adaln_modulate``
(vllm_omni_neuron/diffusion/quantization/adaln_kernels.py:87-201): ``[B, 1, H]`` per batch element, ``[H]`` / ``[1, H]`` shared.

* :func:`sandwich_norm` — forward, differentiable in every tensor.
* :func:`sandwich_norm_bwd` — the gradients themselves.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .adaln import _NORMS

_MAX_HIDDEN = 8192
_MAX_BATCH = 65535
_PER_GATE, _PER_MUL, _PER_ADD = 1, 2, 4  # VOMNI_PER_*


class SandwichGrads(NamedTuple):
    """Gradients in the shapes and dtypes of the tensors they belong to (None where that was None)."""

    x: torch.Tensor | None
    residual: torch.Tensor
    gate: torch.Tensor | None
    mul: torch.Tensor | None
    add: torch.Tensor | None
    post_weight: torch.Tensor | None


def _rows(name: str, t: torch.Tensor, shape) -> torch.Tensor:
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} must be {tuple(shape)}")
    return _lib.dense(t)


def _vector(name: str, v: torch.Tensor, batch: int, hidden: int) -> torch.Tensor:
    """``v`` checked, as dense fp32."""
    shape = v.shape
    if len(shape) == 3 and name != "post_weight":
        if shape != (batch, 1, hidden):
            raise ValueError(f"per-batch {name} must be [{batch}, 1, {hidden}], got {tuple(shape)}")
    elif shape != (hidden,) and shape != (1, hidden):
        raise ValueError(f"{name} must be {'' if name == 'post_weight' else f'[{batch}, 1, {hidden}] or '}[{hidden}], got {tuple(shape)}")
    if v.dtype is not torch.float32:
        if v.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {v.dtype}")
        v = v.float()
    return _lib.dense(v)


def _plan(x, residual, gate, mul, add, post_weight, eps, post_norm, norm_type):
    """Checked ``(hidden, rows, rows_per_mod, per bits, post kind, norm kind, the vectors in fp32)`` of a call."""
    if not 0 < eps < float("inf"):
        raise ValueError(f"eps must be positive and finite, got {eps}")
    if post_norm not in _NORMS:
        raise ValueError(f"unsupported post_norm {post_norm!r}")
    if norm_type not in _NORMS:
        raise ValueError(f"unsupported norm_type {norm_type!r}")
    shape = residual.shape
    if len(shape) < 2:
        raise ValueError("residual must have at least 2 dims")
    hidden = shape[-1]
    if not 0 < hidden <= _MAX_HIDDEN or hidden % 8:
        raise ValueError(f"hidden dim {hidden} unsupported (needs H <= {_MAX_HIDDEN} and H % 8 == 0)")
    if x is None:
        for name, v in (("gate", gate), ("post_weight", post_weight)):
            if v is not None:
                raise ValueError(f"{name} requires x (it scales the sub-layer output)")
    batch = shape[0] if len(shape) == 3 else 1
    rows = residual.numel() // hidden
    bits = 0
    if gate is not None:
        gate = _vector("gate", gate, batch, hidden)
        bits = _PER_GATE if gate.dim() == 3 else 0
    if mul is not None:
        mul = _vector("mul", mul, batch, hidden)
        bits |= _PER_MUL if mul.dim() == 3 else 0
    if add is not None:
        add = _vector("add", add, batch, hidden)
        bits |= _PER_ADD if add.dim() == 3 else 0
    if post_weight is not None:
        post_weight = _vector("post_weight", post_weight, batch, hidden)
    if bits and batch > _MAX_BATCH:
        raise ValueError(f"per-batch vectors of more than {_MAX_BATCH} batch elements are unsupported, got {batch}")
    per_mod = rows // batch if bits and batch else rows
    return hidden, rows, per_mod, bits, _NORMS[post_norm], _NORMS[norm_type], gate, mul, add, post_weight


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, residual, gate, mul, add, post_weight, eps, post_norm, norm_type):
    hidden, rows, per_mod, bits, post, norm, gate, mul, add, post_weight = _plan(x, residual, gate, mul, add, post_weight, eps,
                                                                                 post_norm, norm_type)
    dev = _lib.one_device(x, residual, gate, mul, add, post_weight)
    if x is not None:
        x = _rows("x", x, residual.shape)
    residual = _rows("residual", residual, residual.shape)
    res_out = None if x is None else torch.empty_like(residual)
    out = torch.empty_like(residual)
    if rows:
        _lib.launch(dev, "vomni_sandwich_norm", _ptr(x), residual.data_ptr(), _ptr(gate), _ptr(post_weight), _ptr(mul), _ptr(add), rows,
                    hidden, per_mod, bits, eps, post, norm, _ptr(res_out), out.data_ptr())
    return res_out, out


def _backward(grad_res, grad_out, x, residual_out, gate, mul, add, post_weight, eps, post_norm, norm_type, need):
    """``need``: whether gate's, mul's, add's and post_weight's gradients are asked for."""
    given = (gate, mul, add, post_weight)
    hidden, rows, per_mod, bits, post, norm, *vectors = _plan(x, residual_out, *given, eps, post_norm, norm_type)
    dev = _lib.one_device(grad_res, grad_out, x, residual_out, *vectors)
    shape = residual_out.shape
    if grad_res is not None:
        grad_res = _rows("grad_residual_out", grad_res, shape)
    if grad_out is not None:
        grad_out = _rows("grad_out", grad_out, shape)
    dx = None
    if x is not None:
        x = _rows("x", x, shape)
        dx = torch.empty_like(x)
    residual_out = _rows("residual_out", residual_out, shape)
    dres = torch.empty_like(residual_out)
    make = torch.empty_like if rows else torch.zeros_like
    sums = [make(v) if v is not None and n else None for v, n in zip(vectors, need)]  # fp32 and dense, as the vectors now are
    if rows:
        ws_bytes = _lib.workspace_bytes(dev, "vomni_sandwich_norm", rows, hidden, per_mod)
        ws = _lib.workspace(ws_bytes, residual_out.device)
        gate, mul, _, post_weight = vectors
        dgate, dmul, dadd, dw = map(_ptr, sums)
        _lib.launch(dev, "vomni_sandwich_norm_bwd", _ptr(grad_res), _ptr(grad_out), _ptr(x), residual_out.data_ptr(), _ptr(gate),
                    _ptr(post_weight), _ptr(mul), rows, hidden, per_mod, bits, eps, post, norm, _ptr(dx), dres.data_ptr(), dgate, dw,
                    dmul, dadd, ws.data_ptr(), ws_bytes)
    return SandwichGrads(dx, dres, *(t if t is None or t.dtype is g.dtype else t.to(g.dtype) for t, g in zip(sums, given)))


class _SandwichNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, mul, add, post_weight, eps, post_norm, norm_type):
        ctx.set_materialize_grads(False)
        res_out, out = _forward(x, residual, gate, mul, add, post_weight, eps, post_norm, norm_type)
        ctx.save_for_backward(x, residual if x is None else res_out, gate, mul, add, post_weight)
        ctx.kinds = (eps, post_norm, norm_type)
        return out if x is None else (res_out, out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, res, gate, mul, add, post_weight = ctx.saved_tensors
        grad_res, grad_out = (None, grads[0]) if x is None else grads
        if grad_res is None and grad_out is None:
            return (None,) * 9
        need = ctx.needs_input_grad[:6]
        grads = _backward(grad_res, grad_out, x, res, gate, mul, add, post_weight, *ctx.kinds, need[2:])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def sandwich_norm(
    x: torch.Tensor | None,
    residual: torch.Tensor,
    gate: torch.Tensor | None = None,
    mul: torch.Tensor | None = None,
    add: torch.Tensor | None = None,
    *,
    eps: float,
    post_norm: str = "rms_norm",
    post_weight: torch.Tensor | None = None,
    norm_type: str = "layer_norm",
):
    """``(residual_out, out)`` of ``residual_out = residual + gate * post(x) * post_weight`` and
    ``out = norm(residual_out) * mul + add``; differentiable in every tensor.

    * ``x``, ``residual``: ``[B, S, H]`` or ``[T, H]`` bf16, ``H <= 8192``, ``H % 8 == 0``. ``x=None``: no branch, ``residual_out``
      is ``residual`` itself (``gate`` and ``post_weight`` must be None, ``post_norm`` is ignored).
    * ``gate`` / ``mul`` / ``add``: ``[B, 1, H]`` or ``[H]`` / ``[1, H]`` in fp32, bf16 or fp16, or None (1, 1, 0);
      ``post_weight``: ``[H]``. They are used in fp32.
    * ``post_norm`` / ``norm_type``: ``"layer_norm"``, ``"rms_norm"`` or ``"none"``; ``eps > 0`` is added to both variances.

    Arithmetic is fp32; ``out`` comes from the unrounded residual, and each result is rounded to bf16 once. The backward pass
    reads ``x`` and ``residual_out`` and recomputes the statistics; it gives the same bits every time.
    """
    if _lib.for_autograd(x, residual, gate, mul, add, post_weight):
        res = _SandwichNorm.apply(x, residual, gate, mul, add, post_weight, float(eps), post_norm, norm_type)
        return (residual, res) if x is None else res
    res_out, out = _forward(x, residual, gate, mul, add, post_weight, float(eps), post_norm, norm_type)
    return (residual if x is None else res_out), out


def sandwich_norm_bwd(
    grad_residual_out: torch.Tensor | None,
    grad_out: torch.Tensor | None,
    x: torch.Tensor | None,
    residual_out: torch.Tensor,
    gate: torch.Tensor | None = None,
    mul: torch.Tensor | None = None,
    add: torch.Tensor | None = None,
    *,
    eps: float,
    post_norm: str = "rms_norm",
    post_weight: torch.Tensor | None = None,
    norm_type: str = "layer_norm",
) -> SandwichGrads:
    """Gradients of :func:`sandwich_norm` from those of its two results (one of them may be None: zero), its arguments and
    the ``residual_out`` it returned (``residual`` itself where ``x`` is None). Not differentiable themselves."""
    _lib.refuse_tangents("sandwich_norm_bwd", grad_residual_out, grad_out, x, residual_out, gate, mul, add, post_weight)
    if grad_residual_out is None and grad_out is None:
        raise ValueError("at least one of grad_residual_out and grad_out is needed")
    return _backward(grad_residual_out, grad_out, x, residual_out, gate, mul, add, post_weight, float(eps), post_norm, norm_type,
                     (True,) * 4)
