"""Wan 3-D RoPE tables and the FP8 leaf's weight / cache transforms (torch, host side).

* :func:`wan_rotary_freqs` — ``WanRotaryPosEmbed`` (vllm_omni_neuron/diffusion/layers/rope.py:37-114):
  per-token interleaved ``(cos, sin)`` ``[1, S, 1, head_dim]`` for a ``(frames, height, width)`` latent.
* :func:`apply_rotary_emb_wan` — rope.py:8-34 (interleaved lane pairs).
* :func:`rope_rotate_half_caches` — ``_rope_rotate_half_caches``
  (vllm_omni_neuron/diffusion/quantization/row_mx_modules.py:51-76).
* :func:`deinterleave_perm`, :func:`deinterleave_qk_columns`, :func:`deinterleave_gamma_row` —
  vllm_omni_neuron/diffusion/quantization/row_mx_loaders.py:26-71: the per-head channel permutation
  that lets a rotate-half RoPE reproduce Wan's interleaved RoPE.

On the device, from positions instead of tables:

* :func:`rotary_axes` — rotary positions with several axes for query and key heads, differentiable.
* :func:`wan_grid_positions` — the ``(frame, row, column)`` positions of a latent's patches.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_PAIRINGS = {"interleaved": 0, "half": 1}
_ROTARY_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITION_DTYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def _rope_1d(dim: int, max_seq_len: int, theta: float):
    freqs = 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    t = torch.arange(max_seq_len, dtype=torch.float64)
    f = torch.outer(t, freqs)
    return f.cos().float().repeat_interleave(2, dim=-1), f.sin().float().repeat_interleave(2, dim=-1)


def wan_rotary_freqs(head_dim: int, patch_size, max_seq_len: int, latent_fhw, theta: float = 10000.0, device=None):
    """(cos, sin), each ``[1, S, 1, head_dim]`` fp32, for a latent of ``(frames, height, width)``."""
    h_dim = w_dim = 2 * (head_dim // 6)
    t_dim = head_dim - h_dim - w_dim
    parts = [_rope_1d(d, max_seq_len, theta) for d in (t_dim, h_dim, w_dim)]
    fc = torch.cat([p[0] for p in parts], dim=1)
    fs = torch.cat([p[1] for p in parts], dim=1)
    f, hh, ww = latent_fhw
    pt, ph, pw = patch_size
    ppf, pph, ppw = f // pt, hh // ph, ww // pw
    split = [head_dim - 2 * (head_dim // 3), head_dim // 3, head_dim // 3]
    out = []
    for tab in (fc, fs):
        a, b, c = tab.split(split, dim=1)
        a = a[:ppf].view(ppf, 1, 1, -1).expand(ppf, pph, ppw, -1)
        b = b[:pph].view(1, pph, 1, -1).expand(ppf, pph, ppw, -1)
        c = c[:ppw].view(1, 1, ppw, -1).expand(ppf, pph, ppw, -1)
        out.append(torch.cat([a, b, c], dim=-1).reshape(1, ppf * pph * ppw, 1, -1).to(device))
    return out[0], out[1]


def apply_rotary_emb_wan(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Interleaved RoPE on ``[B, S, H, D]`` (fp32 math, result in x's dtype)."""
    x1, x2 = x.unflatten(-1, (-1, 2)).unbind(-1)
    c = cos[..., 0::2]
    s = sin[..., 1::2]
    return torch.stack((x1 * c - x2 * s, x1 * s + x2 * c), dim=-1).flatten(-2, -1).to(x.dtype)


def rope_rotate_half_caches(cos: torch.Tensor, sin: torch.Tensor):
    """Rotate-half caches ``cat([base, base])`` from interleaved tables (row_mx_modules.py:51-76)."""
    base_cos = cos[..., 0::2]
    base_sin = sin[..., 1::2]
    return torch.cat([base_cos, base_cos], dim=-1), torch.cat([base_sin, base_sin], dim=-1)


def deinterleave_perm(head_dim: int) -> torch.Tensor:
    if head_dim % 2:
        raise ValueError(f"head_dim must be even for interleaved RoPE, got {head_dim}")
    idx = torch.arange(head_dim // 2)
    return torch.cat([2 * idx, 2 * idx + 1])


def deinterleave_qk_columns(t: torch.Tensor, q_size: int, kv_size: int, head_dim: int) -> torch.Tensor:
    perm = deinterleave_perm(head_dim).to(t.device)
    q_idx = torch.arange(q_size, device=t.device).reshape(-1, head_dim)[:, perm].flatten()
    k_idx = q_size + torch.arange(kv_size, device=t.device).reshape(-1, head_dim)[:, perm].flatten()
    v_idx = torch.arange(q_size + kv_size, t.shape[-1], device=t.device)
    return t.index_select(-1, torch.cat((q_idx, k_idx, v_idx)))


def deinterleave_gamma_row(gamma: torch.Tensor, head_dim: int) -> torch.Tensor:
    perm = deinterleave_perm(head_dim).to(gamma.device)
    n = gamma.numel() // head_dim
    return gamma.reshape(n, head_dim).index_select(-1, perm).reshape(1, n * head_dim)


# ---------------------------------------------------------------- rotary positions with several axes


def wan_grid_positions(latent_fhw, patch_size=(1, 2, 2), device=None) -> torch.Tensor:
    """``[S, 3]`` int32 ``(frame, row, column)`` of every patch of a ``(frames, height, width)`` latent, in the token
    order of :func:`wan_rotary_freqs`."""
    f, h, w = (n // p for n, p in zip(latent_fhw, patch_size))
    i = torch.arange(f * h * w, dtype=torch.int32, device=device)
    return torch.stack([i // (h * w), i // max(w, 1) % max(h, 1), i % max(w, 1)], dim=-1)


def _rotary_source(t: torch.Tensor):
    """(tensor, row stride, batch stride) as the kernel reads it: heads dense inside a token, strides of 16 bytes
    (column slices of a fused projection pass as they are); anything else is copied."""
    b, s, h, d = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, h * d, s * h * d
    sb, ss, sh, sd = t.stride()
    row, batch = ss if s > 1 else h * d, sb if b > 1 else s * h * d
    unit = 16 // t.element_size()
    if (sd == 1 and (h == 1 or sh == d) and row >= h * d and batch >= 0 and row % unit == 0 and batch % unit == 0
            and t.data_ptr() % 16 == 0):
        return t, row, batch
    return _lib.dense(t), h * d, s * h * d


def _rotary(q, k, positions, axes_dims, theta, pairing, inverse):
    b, s, hq, d = q.shape
    q_out = k_out = None
    q_args = k_args = (None, None, 0, 0, 0)
    if q.numel():
        q, row, batch = _rotary_source(q)
        q_out = _lib.empty(q)
        q_args = (q.data_ptr(), q_out.data_ptr(), hq, row, batch)
    if k is not None and k.numel():
        k, row, batch = _rotary_source(k)
        k_out = _lib.empty(k)
        k_args = (k.data_ptr(), k_out.data_ptr(), k.shape[2], row, batch)
    if q_out is not None or k_out is not None:
        if not positions.is_contiguous():
            positions = positions.contiguous()
        n = len(axes_dims)
        _lib.launch(q.get_device(), "vomni_rotary_axes", *q_args, *k_args, b, s, d, positions.data_ptr(),
                    _POSITION_DTYPES[positions.dtype], int(positions.dim() == 3), n, (ctypes.c_int * n)(*axes_dims), theta, pairing,
                    int(inverse), _ROTARY_DTYPES[q.dtype])
    if q_out is None:
        q_out = q.new_empty(q.shape)
    if k_out is None and k is not None:
        k_out = k.new_empty(k.shape)
    return q_out, k_out


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes_dims, theta, pairing, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rest = (axes_dims, theta, pairing, inverse)
        return _rotary(q, k, positions, axes_dims, theta, pairing, inverse)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        axes_dims, theta, pairing, inverse = ctx.rest
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is None and gk is None:
            return (None,) * 7
        first, second = (gq, gk) if gq is not None else (gk, None)
        out = _rotary(first, second, positions, axes_dims, theta, pairing, not inverse)
        dq, dk = out if gq is not None else (None, out[0])
        return dq, dk, None, None, None, None, None


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes_dims, *, theta: float = 10000.0,
                pairing: str = "interleaved", inverse: bool = False):
    """Rotary positions with several axes, for query and key heads in one pass; differentiable in ``q`` and ``k``.

    A head's ``d`` values are ``d / 2`` pairs, axis ``a`` owning the next ``axes_dims[a] / 2``; its pair ``i`` turns by
    ``positions[..., a] * theta ** (-2 i / axes_dims[a])``. ``axes_dims=(44, 42, 42)`` with interleaved pairs is Wan's
    rotary embedding (``WanRotaryPosEmbed`` + ``apply_rotary_emb_wan``, vllm_omni_neuron/diffusion/layers/rope.py:8-114).

    * ``q [b, s, hq, d]``, ``k [b, s, hk, d]`` (or None) token-major, bf16 / fp16 / fp32, ``d % 16 == 0``, ``d <= 256``; the
      column slices of a fused projection are read in place, other strides are copied first.
    * ``positions`` ``[s, n_axes]`` or ``[b, s, n_axes]``, int32 / int64 / fp32 (fractions for interpolated positions).
      Angles are formed and reduced in 64 bits, so they are off by some 2^-52 of their size: less than fp32 holds of
      the reduced angle up to positions of 10^8. Not differentiated.
    * ``pairing``: ``"interleaved"`` pairs values ``(2p, 2p + 1)``, ``"half"`` pairs ``(p, p + d / 2)``.
    * ``inverse`` turns by the negative angles (what the gradient does).

    Returns ``(q', k')``, dense tensors of the inputs' dtype (``q'`` alone when ``k`` is None); fp32 arithmetic, rounded once.
    """
    if pairing not in _PAIRINGS:
        raise ValueError(f"unknown pairing {pairing!r}")
    axes_dims = tuple(map(int, axes_dims))
    for name, t in (("q", q),) if k is None else (("q", q), ("k", k)):
        if len(t.shape) != 4:
            raise ValueError(f"{name} must be token-major [b, s, heads, d], got {tuple(t.shape)}")
        if t.dtype not in _ROTARY_DTYPES:
            raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    b, s, _, d = q.shape
    if k is not None:
        kb, ks, _, kd = k.shape
        if kb != b or ks != s or kd != d:
            raise ValueError(f"k {tuple(k.shape)} must match q {tuple(q.shape)} but for the heads")
        if k.dtype is not q.dtype:
            raise TypeError(f"q and k must have one dtype, got {q.dtype} and {k.dtype}")
    if d % 16 or not 0 < d <= 256:
        raise ValueError(f"head dim {d} unsupported (needs d % 16 == 0 and d <= 256)")
    if not 1 <= len(axes_dims) <= 4 or min(axes_dims) <= 0 or sum(axes_dims) != d or [n for n in axes_dims if n % 2]:
        raise ValueError(f"axes_dims {axes_dims} must be 1 to 4 even counts that sum to the head dim {d}")
    if positions.dtype not in _POSITION_DTYPES:
        raise TypeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.shape not in ((s, len(axes_dims)), (b, s, len(axes_dims))):
        raise ValueError(f"positions must be [{s}, {len(axes_dims)}] or [{b}, {s}, {len(axes_dims)}], got {tuple(positions.shape)}")
    if not (theta > 0 and theta < float("inf")):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    _lib.one_device(q, k, positions)
    args = (q, k, positions, axes_dims, float(theta), _PAIRINGS[pairing], bool(inverse))
    if _lib.for_autograd(q, k):
        out = _RotaryAxes.apply(*args)
    else:
        out = _rotary(*args)
    return out[0] if k is None else out
