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
_PER = {"gate": 1, "mul": 2, "add": 4}  # VOMNI_PER_*


class SandwichGrads(NamedTuple):
    """Gradients in the shapes and dtypes of the tensors they belong to (None where that was None)."""

    x: torch.Tensor | None
    residual: torch.Tensor
    gate: torch.Tensor | None
    mul: torch.Tensor | None
    add: torch.Tensor | None
    post_weight: torch.Tensor | None


def _rows(name: str, t: torch.Tensor, shape) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} must be {tuple(shape)}")
    return _lib.dense(t)


def _vector(name: str, v: torch.Tensor | None, batch: int, hidden: int):
    """(fp32 dense rows or None, whether one per batch element)."""
    if v is None:
        return None, False
    if v.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {v.dtype}")
    shape = v.shape
    if len(shape) == 3 and name != "post_weight":
        if shape != (batch, 1, hidden):
            raise ValueError(f"per-batch {name} must be [{batch}, 1, {hidden}], got {tuple(shape)}")
        per = True
    elif shape != (hidden,) and shape != (1, hidden):
        raise ValueError(f"{name} must be {'' if name == 'post_weight' else f'[{batch}, 1, {hidden}] or '}[{hidden}], got {tuple(shape)}")
    else:
        per = False
    return _lib.dense(v if v.dtype == torch.float32 else v.float()), per


def _plan(x, residual, vectors, eps, post_norm, norm_type):
    """Checked (hidden, rows, rows_per_mod, per bits, fp32 vectors) of a call."""
    if not 0 < eps < float("inf"):
        raise ValueError(f"eps must be positive and finite, got {eps}")
    if post_norm not in _NORMS:
        raise ValueError(f"unsupported post_norm {post_norm!r}")
    if norm_type not in _NORMS:
        raise ValueError(f"unsupported norm_type {norm_type!r}")
    if residual.dim() < 2:
        raise ValueError("residual must have at least 2 dims")
    hidden = residual.shape[-1]
    if not 0 < hidden <= _MAX_HIDDEN or hidden % 8:
        raise ValueError(f"hidden dim {hidden} unsupported (needs H <= {_MAX_HIDDEN} and H % 8 == 0)")
    if x is None:
        for name in ("gate", "post_weight"):
            if vectors[name] is not None:
                raise ValueError(f"{name} requires x (it scales the sub-layer output)")
    batch = residual.shape[0] if residual.dim() == 3 else 1
    rows = residual.numel() // hidden
    dense, bits = {}, 0
    for name, v in vectors.items():
        dense[name], per = _vector(name, v, batch, hidden)
        bits |= _PER[name] if per else 0
    if bits and batch > _MAX_BATCH:
        raise ValueError(f"per-batch vectors of more than {_MAX_BATCH} batch elements are unsupported, got {batch}")
    return hidden, rows, rows // batch if bits and batch else rows, bits, dense


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _forward(x, residual, gate, mul, add, post_weight, eps, post_norm, norm_type):
    hidden, rows, per_mod, bits, v = _plan(
        x, residual, {"gate": gate, "mul": mul, "add": add, "post_weight": post_weight}, eps, post_norm, norm_type)
    dev = _lib.one_device(x, residual, gate, mul, add, post_weight)
    x = None if x is None else _rows("x", x, residual.shape)
    residual = _rows("residual", residual, residual.shape)
    res_out = None if x is None else residual.new_empty(residual.shape)
    out = residual.new_empty(residual.shape)
    if rows:
        _lib.launch(dev, "vomni_sandwich_norm", _ptr(x), residual.data_ptr(), _ptr(v["gate"]), _ptr(v["post_weight"]), _ptr(v["mul"]),
                    _ptr(v["add"]), rows, hidden, per_mod, bits, eps, _NORMS[post_norm], _NORMS[norm_type], _ptr(res_out),
                    out.data_ptr())
    return res_out, out


def _backward(grad_res, grad_out, x, residual_out, gate, mul, add, post_weight, eps, post_norm, norm_type, need):
    vectors = {"gate": gate, "mul": mul, "add": add, "post_weight": post_weight}
    hidden, rows, per_mod, bits, v = _plan(x, residual_out, vectors, eps, post_norm, norm_type)
    dev = _lib.one_device(grad_res, grad_out, x, residual_out, *vectors.values())
    shape = residual_out.shape
    grad_res = None if grad_res is None else _rows("grad_residual_out", grad_res, shape)
    grad_out = None if grad_out is None else _rows("grad_out", grad_out, shape)
    x = None if x is None else _rows("x", x, shape)
    residual_out = _rows("residual_out", residual_out, shape)
    dx = None if x is None else x.new_empty(shape)
    dres = residual_out.new_empty(shape)
    make = residual_out.new_empty if rows else residual_out.new_zeros
    sums = {n: make(t.shape, dtype=torch.float32) if t is not None and need[n] else None for n, t in vectors.items()}
    if rows:
        ws_bytes = _lib.on_device(dev, _lib.load().vomni_sandwich_norm_workspace_bytes, rows, hidden, per_mod)
        ws = residual_out.new_empty(ws_bytes, dtype=torch.uint8)
        _lib.launch(dev, "vomni_sandwich_norm_bwd", _ptr(grad_res), _ptr(grad_out), _ptr(x), residual_out.data_ptr(), _ptr(v["gate"]),
                    _ptr(v["post_weight"]), _ptr(v["mul"]), rows, hidden, per_mod, bits, eps, _NORMS[post_norm], _NORMS[norm_type],
                    _ptr(dx), dres.data_ptr(), _ptr(sums["gate"]), _ptr(sums["post_weight"]), _ptr(sums["mul"]), _ptr(sums["add"]),
                    ws.data_ptr(), ws_bytes)
    done = {n: t if t is None or vectors[n].dtype == torch.float32 else t.to(vectors[n].dtype) for n, t in sums.items()}
    return SandwichGrads(dx, dres, done["gate"], done["mul"], done["add"], done["post_weight"])


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
        names = ("x", "residual", "gate", "mul", "add", "post_weight")
        need = dict(zip(names, ctx.needs_input_grad))
        g = _backward(grad_res, grad_out, x, res, gate, mul, add, post_weight, *ctx.kinds, need)
        return tuple(getattr(g, n) if need[n] else None for n in names) + (None, None, None)


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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, gate, mul, add, post_weight)):
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
    the ``residual_out`` it returned (``residual`` itself where ``x`` is None)."""
    if grad_residual_out is None and grad_out is None:
        raise ValueError("at least one of grad_residual_out and grad_out is needed")
    need = dict.fromkeys(("gate", "mul", "add", "post_weight"), True)
    return _backward(grad_residual_out, grad_out, x, residual_out, gate, mul, add, post_weight, float(eps), post_norm, norm_type,
                     need)
