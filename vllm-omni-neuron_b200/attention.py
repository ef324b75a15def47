"""Const-max (ring) attention: the reference's kernel-call API and attention processor on B200.

* :func:`ring_attention_const_max_fwd` keeps the signature and return contract of the NKI kernel
  (vllm_omni_neuron/kernels/nkilib/experimental/attention/ring_attention_const_max_fwd.py:958-1017):
  token-major ``q, k, v [b, S_loc, h, 128]`` bf16 in, head-major ``o [b, h, S_loc, 128]`` out
  (plus ``lse [b, h, 128, ceil(S_loc/128)]`` fp32 when ``training``); ``softmax_scale`` defaults
  to ``1/sqrt(d)``; ``kv_prefetch_depth`` is clamped to ``[1, num_workers-1]``; shape contract
  violations raise ``AssertionError`` as the kernel's ``kernel_assert`` does (:1019-1031).
* :func:`wan_cp_self_attention` keeps the attention-processor signature
  (vllm_omni_neuron/diffusion/models/wan2_2/wan2_2_transformer.py:806-847) and returns the d-major
  ``[B, N, D, S_loc]`` layout directly from the kernel epilogue (the reference transposes after the
  kernel, :836).

All compute runs in ``libvomni_b200.so`` (sm_100a). There is no fallback path: a missing library or
a non-sm_100 device raises.

Host-resident inputs (B200 extension): when q, k and v are pinned CPU tensors, both entry points
stream them to the current CUDA device in head groups — the copy of group i+1 (copy engine, 2-D
strided copies straight out of the token-major host layout) overlaps the attention of group i, and
the result of group i returns to pinned host memory while group i+1 computes. Heads are
independent, so the result is identical to the device-resident call; the output is a pinned CPU
tensor, complete on return.

Training: :func:`attention_fwd` (output and log-sum-exp; keys of another sequence, shared key heads and uneven batches
included) is differentiable through :func:`attention_bwd` (the gradients); :func:`wan_attention` is its output alone.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_HEAD_DIM = 128


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q, k, v must be token-major [b, seqlen, h, d]"
    b, s, h, d = q.shape
    assert k.shape[2] == h, "expects q_heads == kv_heads, broadcast before calling"
    assert d == _HEAD_DIM, f"head_dim must be 128, got {d}"
    assert tuple(k.shape) == (b, s, h, d) and tuple(v.shape) == (b, s, h, d), (
        f"q and k must be token-major [b, seqlen, h, d]; got q={tuple(q.shape)}, k={tuple(k.shape)}"
    )
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor (the B200 kernel has no CPU path)")
    return b, s, h, d


def token_major(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, token stride in elements) for a token-major ``[b, s, h, d]`` view.

    Views whose heads are dense inside a token row (for example the Q/K/V column slices of a fused
    ``[b, s, 3*h*d]`` projection, ``tensor_split`` in row_mx_modules.py:390) are passed through with
    their row stride; anything else is made contiguous."""
    b, s, h, d = t.shape
    st = t.stride()
    ok = (
        st[3] == 1 and st[2] == d and st[1] >= h * d and st[1] % 8 == 0
        and (b == 1 or st[0] == s * st[1]) and t.data_ptr() % 16 == 0
    )
    if ok:
        return t, st[1]
    return t.contiguous(), h * d


_HOST_GROUP_HEADS = 5


def _host_group_heads(s: int, h: int, dev: torch.device, world: int = 1) -> int:
    """Heads per host-streamed group. One rank (PCIe-bound, cheap calls): 5, the finest split that
    measured fastest. A CP ring (every call pays an all-reduce, block copies and several pass
    launches): the finest split whose passes still fill two waves of CTA pairs (a pair covers 512
    query rows of one head on two SMs), e.g. 20 heads for S_loc = 4095, 10 for 8190."""
    if world <= 1:
        return min(h, _HOST_GROUP_HEADS)
    pairs_per_head = -(-s // 512)
    slots = max(1, torch.cuda.get_device_properties(dev).multi_processor_count // 2)
    g_min = max(_HOST_GROUP_HEADS, -(-2 * slots // pairs_per_head))
    groups = max(1, h // g_min)
    return -(-h // groups)
_AUX_STREAMS: dict = {}


def _aux_streams(dev: torch.device):
    """(host->device copy stream, device->host copy stream, second compute stream) of a device."""
    key = dev.index
    if key not in _AUX_STREAMS:
        _AUX_STREAMS[key] = tuple(torch.cuda.Stream(dev) for _ in range(3))
    return _AUX_STREAMS[key]


def _copy_2d(dst_ptr, dpitch, src_ptr, spitch, width, height, stream):
    _lib.check(_lib.load().vomni_memcpy_2d_async(dst_ptr, dpitch, src_ptr, spitch, width, height, stream.cuda_stream),
               "vomni_memcpy_2d_async")


def _host_streamed(fn, q, k, v, *, out_layout: str, training: bool, alternate: bool = True,
                   group_heads: int | None = None, world: int = 1):
    """Run ``fn(q_dev, k_dev, v_dev) -> out | (out, lse)`` over head groups of pinned host q/k/v
    (``group_heads`` heads per group, default ``_host_group_heads`` for a ring of ``world`` ranks).

    Group g's host->device copies run on a copy stream, its attention alternates between the
    caller's stream and a second compute stream (so one group's tail wave overlaps the next group;
    ``alternate=False`` keeps every group on the caller's stream, as a ring context's buffers
    require), and its output returns on a second copy stream. Returns pinned host tensors."""
    b, s, h, d = q.shape
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.device.type != "cpu" or not t.is_pinned():
            raise ValueError(f"host-resident {name} must be a pinned CPU tensor (tensor.pin_memory())")
        if t.dtype != torch.bfloat16 or tuple(t.shape) != (b, s, h, d):
            raise TypeError(f"{name} must be bfloat16 [b, s, h, d] like q")
    q, k, v = (t if t.is_contiguous() else t.contiguous().pin_memory() for t in (q, k, v))
    dev = torch.device("cuda", torch.cuda.current_device())
    main = torch.cuda.current_stream(dev)
    h2d, d2h, alt = _aux_streams(dev)
    esz = 2
    dq, dk, dv = (torch.empty((b, s, h, d), dtype=torch.bfloat16, device=dev) for _ in range(3))
    o_shape = (b, h, d, s) if out_layout == "bhds" else (b, h, s, d)
    host_o = torch.empty(o_shape, dtype=torch.bfloat16, pin_memory=True)
    n_lse = 128 * (-(-s // 128))
    host_lse = torch.empty((b, h, 128, n_lse // 128), dtype=torch.float32, pin_memory=True) if training else None
    gh = max(1, int(group_heads or _host_group_heads(s, h, dev, world)))
    row = h * d * esz
    h2d.wait_stream(main)
    alt.wait_stream(main)
    keep = []
    for gi, h0 in enumerate(range(0, h, gh)):
        h1 = min(h, h0 + gh)
        w = (h1 - h0) * d * esz
        for src, dst in ((q, dq), (k, dk), (v, dv)):
            _copy_2d(dst.data_ptr() + h0 * d * esz, row, src.data_ptr() + h0 * d * esz, row, w, b * s, h2d)
        arrived = torch.cuda.Event()
        arrived.record(h2d)
        cs = alt if (alternate and gi % 2) else main
        cs.wait_event(arrived)
        with torch.cuda.stream(cs):
            res = fn(dq[:, :, h0:h1], dk[:, :, h0:h1], dv[:, :, h0:h1])
        o, lse = res if training else (res, None)
        done = torch.cuda.Event()
        done.record(cs)
        d2h.wait_event(done)
        per_head = o[0, 0].numel() * esz
        _copy_2d(host_o.data_ptr() + h0 * per_head, h * per_head, o.data_ptr(), (h1 - h0) * per_head,
                 (h1 - h0) * per_head, b, d2h)
        if training:
            lh = 128 * (n_lse // 128) * 4
            _copy_2d(host_lse.data_ptr() + h0 * lh, h * lh, lse.data_ptr(), (h1 - h0) * lh, (h1 - h0) * lh, b, d2h)
        keep.append(res)
    d2h.synchronize()  # every group's copy-out waited for its compute, which waited for its copy-in
    main.wait_stream(alt)
    main.wait_stream(d2h)
    del keep
    return (host_o, host_lse) if training else host_o


def _stream_ptr(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def attention_local(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    softmax_scale: float | None = None,
    *,
    out_layout: str = "bhsd",
    training: bool = False,
):
    """Single-rank const-max attention (``num_workers == 1``): prologue norms + one final pass.

    ``out_layout``: ``"bhsd"`` (kernel layout) or ``"bhds"`` (d-major, the attention-processor
    layout). Returns ``o`` or ``(o, lse)``.
    """
    b, s, h, d = _check_qkv(q, k, v)
    q, q_stride = token_major(q)
    k, k_stride = token_major(k)
    v, v_stride = token_major(v)
    if k_stride != v_stride:  # K and V share one stride argument
        k, v = k.contiguous(), v.contiguous()
        k_stride = h * d
    scale = float(softmax_scale) if softmax_scale else 1.0 / math.sqrt(d)
    lib = _lib.load()
    flags = 0
    if out_layout == "bhds":
        flags |= _lib.CM_OUT_DMAJOR
        out = torch.empty((b, h, d, s), dtype=torch.bfloat16, device=q.device)
    elif out_layout == "bhsd":
        out = torch.empty((b, h, s, d), dtype=torch.bfloat16, device=q.device)
    else:
        raise ValueError(f"unknown out_layout {out_layout!r}")
    lse = None
    if training:
        flags |= _lib.CM_LSE
        lse = torch.zeros((b, h, 128, -(-s // 128)), dtype=torch.float32, device=q.device)
    ws_bytes = lib.vomni_cm_workspace_bytes(b, s, h, d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    rc = lib.vomni_cm_attention_local_strided(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
        b, s, h, d, q_stride, k_stride, scale, flags, ws.data_ptr(), ws_bytes, _stream_ptr(q.device),
    )
    _lib.check(rc, "vomni_cm_attention_local_strided")
    return (out, lse) if training else out


def ring_attention_const_max_fwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    replica_groups: tuple | None = None,
    num_workers: int = 1,
    softmax_scale: float | None = None,
    training: bool = False,
    lse_dtype: torch.dtype = torch.float32,
    kv_prefetch_depth: int = 2,
    *,
    group=None,
    out_layout: str = "bhsd",
):
    """Fixed-max ring attention forward (non-causal); see the module docstring for the contract.

    ``group`` (B200 addition): the ``torch.distributed`` process group of this rank's ring when
    ``num_workers > 1``; defaults to the group matching ``replica_groups`` (built once per ring).
    Pinned host q/k/v are streamed by head groups (module docstring) and give host results.
    """
    if q.device.type == "cpu" and k.device.type == "cpu" and v.device.type == "cpu":
        assert q.dim() == 4 and q.shape[-1] == _HEAD_DIM, "q, k, v must be token-major [b, seqlen, h, 128]"

        def dev_call(qd, kd, vd):
            return ring_attention_const_max_fwd(qd, kd, vd, replica_groups, num_workers, softmax_scale, training,
                                                torch.float32, kv_prefetch_depth, group=group, out_layout=out_layout)

        res = _host_streamed(dev_call, q, k, v, out_layout=out_layout, training=training, alternate=num_workers <= 1,
                             world=num_workers)
        return (res[0], res[1].to(lse_dtype)) if training else res
    _check_qkv(q, k, v)
    if num_workers <= 1:
        res = attention_local(q, k, v, softmax_scale, out_layout=out_layout, training=training)
    else:
        from .ring import ring_attention

        res = ring_attention(
            q, k, v, replica_groups=replica_groups, num_workers=num_workers, softmax_scale=softmax_scale,
            training=training, kv_prefetch_depth=kv_prefetch_depth, group=group, out_layout=out_layout,
        )
    if training:
        o, lse = res
        return o, lse.to(lse_dtype)
    return res


def wan_cp_self_attention(query, key, value, scale, cp_size, cp_group, cp_replica_groups):
    """Context-parallel self-attention core (wan2_2_transformer.py:806-847).

    ``query/key/value``: token-major ``[B, local_S, N, D]`` bf16. Returns d-major ``[B, N, D, local_S]``.
    ``cp_group``: a ``torch.distributed`` ProcessGroup, or an object exposing one as
    ``device_group`` (vLLM's GroupCoordinator), or None when ``cp_size == 1``. The ring kernel runs at
    every ``cp_size`` (``num_workers=1`` included); there is no all-gather fallback.
    """
    group = getattr(cp_group, "device_group", cp_group)
    return ring_attention_const_max_fwd(
        query, key, value, replica_groups=cp_replica_groups, num_workers=int(cp_size), softmax_scale=scale,
        group=group, out_layout="bhds",
    )


# ---------------------------------------------------------------- training


def _lens(name: str, lens, b: int, s: int):
    """Host token counts per batch element, or None."""
    if lens is None:
        return None
    if isinstance(lens, torch.Tensor):
        raise TypeError(f"{name} must be a sequence of {b} ints on the host (they size the launch), got a tensor")
    lens = [int(n) for n in lens]
    if len(lens) != b or any(not 0 <= n <= s for n in lens):
        raise ValueError(f"{name} must be {b} counts between 0 and {s}, got {lens}")
    return lens


def _training_scale(softmax_scale, signed: bool = False) -> float:
    scale = 1.0 / math.sqrt(_HEAD_DIM) if softmax_scale is None else float(softmax_scale)
    if not 1e-20 <= (abs(scale) if signed else scale) <= 1e20:  # the forward's softmax bound needs a positive one
        raise ValueError(f"softmax_scale must be {'nonzero' if signed else 'positive'} and finite (1e-20 to 1e20), got {scale}")
    return scale


def _check_training(q, k, v, q_lens, kv_lens):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if len(t.shape) != 4:
            raise ValueError(f"{name} must be token-major [b, s, heads, {_HEAD_DIM}], got {tuple(t.shape)}")
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    b, sq, hq, d = q.shape
    kb, skv, hkv, kd = k.shape
    if d != _HEAD_DIM:
        raise ValueError(f"head_dim must be {_HEAD_DIM}, got {d}")
    if k.shape != v.shape or kb != b or kd != d:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [{b}, s_kv, heads, {d}]")
    if hkv == 0 or hq % hkv:
        raise ValueError(f"query heads ({hq}) must be a multiple of key heads ({hkv})")
    return b, sq, skv, hq, hkv, _lens("q_lens", q_lens, b, sq), _lens("kv_lens", kv_lens, b, skv)


def _cross_fwd(q, k, v, scale):
    """(o [b, h, s_q, d], lse) of whole sequences with equal head counts."""
    b, sq, h, d = q.shape
    skv = k.shape[1]
    q, qs = token_major(q)
    k, ks = token_major(k)
    v, vs = token_major(v)
    if ks != vs:
        k, v = k.contiguous(), v.contiguous()
        ks = h * d
    lib = _lib.load()
    o = torch.empty((b, h, sq, d), dtype=torch.bfloat16, device=q.device)
    lse = torch.full((b, h, 128, -(-sq // 128)), -math.inf, dtype=torch.float32, device=q.device)
    ws_bytes = lib.vomni_cm_workspace_bytes(b, sq, h, d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    rc = lib.vomni_attention_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), b, sq, skv, h, d, qs, ks, scale,
                                 ws.data_ptr(), ws_bytes, _stream_ptr(q.device))
    _lib.check(rc, "vomni_attention_fwd")
    return o, lse


def _attention(q, k, v, scale, q_lens, kv_lens):
    """:func:`attention_fwd` of checked arguments."""
    b, sq, hq, _ = q.shape
    skv, hkv = k.shape[1:3]
    dev = _lib.one_device(q, k, v)
    device = q.device
    q, k, v = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (q, k, v))
    with torch.cuda.device(dev):
        if hkv != hq:
            k, v = (t.repeat_interleave(hq // hkv, dim=2) for t in (k, v))
        if q_lens is None and kv_lens is None and b * sq * hq and skv:
            return _cross_fwd(q, k, v, scale)
        o = torch.zeros((b, hq, sq, _HEAD_DIM), dtype=torch.bfloat16, device=device)
        lse = torch.full((b, hq, 128, -(-sq // 128)), -math.inf, dtype=torch.float32, device=device)
        for i in range(b):
            m, n = q_lens[i] if q_lens else sq, kv_lens[i] if kv_lens else skv
            if m and n and hq:
                oi, li = _cross_fwd(q[i : i + 1, :m], k[i : i + 1, :n], v[i : i + 1, :n], scale)
                o[i, :, :m] = oi[0]
                lse[i, :, :, : li.shape[-1]] = li[0]
        return o, lse


class _AttentionFwd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, q_lens, kv_lens):
        ctx.set_materialize_grads(False)
        o, lse = _attention(q, k, v, scale, q_lens, kv_lens)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.rest = (scale, q_lens, kv_lens)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_o, grad_lse):
        if grad_o is None and grad_lse is None:
            return (None,) * 6
        scale, q_lens, kv_lens = ctx.rest
        q, k, v, o, lse = ctx.saved_tensors
        if grad_o is None:
            grad_o = torch.zeros_like(o)
        grads = attention_bwd(grad_o, q, k, v, o, lse, scale, q_lens=q_lens, kv_lens=kv_lens, grad_lse=grad_lse)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None, None, None)


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None, *, q_lens=None,
                  kv_lens=None):
    """``(o [b, hq, s_q, 128] bf16, lse [b, hq, 128, ceil(s_q / 128)] fp32)`` of ``softmax(softmax_scale q k^T) v``.

    ``q [b, s_q, hq, 128]``, ``k, v [b, s_kv, hkv, 128]`` token-major bf16, ``hq % hkv == 0`` (query head ``h`` reads key head
    ``h // (hq // hkv)``). ``lse[.., r, g]`` belongs to token ``128 g + r``, as in :func:`ring_attention_const_max_fwd`.
    ``q_lens`` / ``kv_lens``: tokens of each batch element (host ints); rows behind them are not read, and their output
    is 0 with an lse of -inf, as is that of rows without keys. ``softmax_scale`` (positive) defaults to ``1 / sqrt(128)``.
    Rows sum under the bound ``softmax_scale * |q_i| * max_j |k_j|`` as in :func:`ring_attention_const_max_fwd`; those whose
    probabilities under it are not representable are computed again under their own maximum.
    Differentiable through both results, by :func:`attention_bwd`. ``b * hq`` is at most 8192, per element where lengths are given.
    """
    *_, q_lens, kv_lens = _check_training(q, k, v, q_lens, kv_lens)
    args = (q, k, v, _training_scale(softmax_scale), q_lens, kv_lens)
    return _AttentionFwd.apply(*args) if _lib.for_autograd(q, k, v) else _attention(*args)


_Strides = ctypes.c_longlong * 15  # (token, head, batch) of q, k, v, grad_o, o


def _any_strides(t: torch.Tensor, head_major: bool = False):
    """(tensor, its token, head and batch strides): ``t`` as it is where TMA can address its strides (d dense, the others
    positive multiples of 8), else a copy. ``head_major``: ``t`` is ``[b, heads, s, d]``."""
    st = t.stride()
    ok = t.data_ptr() % 16 == 0
    if ok and not t.is_contiguous():
        sh = t.shape
        ok = st[3] == 1 and all(sh[i] == 1 or (st[i] > 0 and st[i] % 8 == 0) for i in range(3))
    if not ok:
        t = _lib.dense(t)
        st = t.stride()
    return t, ((st[2], st[1], st[0]) if head_major else (st[1], st[2], st[0]))


def attention_bwd(grad_o: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                  softmax_scale: float | None = None, *, q_lens=None, kv_lens=None, grad_lse: torch.Tensor | None = None):
    """``(dq, dk, dv)``, dense bf16 in the shapes of ``q, k, v``, of the attention whose output and log-sum-exp are ``o``, ``lse``.

    ``o`` / ``grad_o [b, hq, s_q, 128]`` bf16 (any strides) and ``lse`` as :func:`attention_fwd` or
    ``ring_attention_const_max_fwd(training=True)`` return them, ``grad_lse`` (None: 0) the gradient of ``lse`` where that was
    used too, as when parts are merged by it; the other arguments as in :func:`attention_fwd`. The
    probabilities are recomputed as ``exp(softmax_scale q k^T - lse)``, so with the ``lse`` and ``o`` of a whole sequence
    and a part of its keys the result is that part's share of the gradients (for a context-parallel ring: the parts'
    ``dq`` add up). ``lse`` has to be that of a softmax: :func:`attention_fwd`'s is, ``ring_attention_const_max_fwd``'s where
    no row's largest score lies more than about 50 below its bound ``softmax_scale * |q_i| * max_j |k_j|``. Rows behind
    ``q_lens`` / ``kv_lens`` are not read and get zero gradients; a row whose lse is -inf has probabilities 0 and no
    ``grad_lse`` (its ``grad_o`` has to be finite all the same). The same call gives the same bits (no atomics). Not differentiable themselves.
    """
    _lib.refuse_tangents("attention_bwd", grad_o, q, k, v, o, lse, grad_lse)
    b, sq, skv, hq, hkv, q_lens, kv_lens = _check_training(q, k, v, q_lens, kv_lens)
    for name, t in (("grad_o", grad_o), ("o", o)):
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        if t.shape != (b, hq, sq, _HEAD_DIM):
            raise ValueError(f"{name} must be [{b}, {hq}, {sq}, {_HEAD_DIM}], got {tuple(t.shape)}")
    if not lse.is_floating_point() or lse.shape != (b, hq, 128, -(-sq // 128)):
        raise ValueError(f"lse must be [{b}, {hq}, 128, {-(-sq // 128)}], got {lse.dtype} {tuple(lse.shape)}")
    if grad_lse is not None and (not grad_lse.is_floating_point() or grad_lse.shape != lse.shape):
        raise ValueError(f"grad_lse must be {list(lse.shape)} like lse, got {grad_lse.dtype} {tuple(grad_lse.shape)}")
    scale = _training_scale(softmax_scale, signed=True)
    dev = _lib.one_device(grad_o, q, k, v, o, lse, grad_lse)
    empty = not (b and sq and skv and hq)
    if empty:
        return tuple(t.new_zeros(t.shape) for t in (q, k, v))
    dq, dk, dv = _lib.empty(q), _lib.empty(k), _lib.empty(v)
    q, q_st = _any_strides(q)
    k, k_st = _any_strides(k)
    v, v_st = _any_strides(v)
    grad_o, go_st = _any_strides(grad_o, True)
    o, o_st = _any_strides(o, True)
    strides = _Strides(*q_st, *k_st, *v_st, *go_st, *o_st)
    lse = _lib.dense(lse.float())
    if grad_lse is not None:
        grad_lse = _lib.dense(grad_lse.float())
    if q_lens is None and kv_lens is None:
        ws_bytes = _lib.workspace_bytes(dev, "vomni_attention_bwd", b, sq, skv, hq, hkv, _HEAD_DIM, None, None)
    else:
        q_lens, kv_lens = (n if n is None else (ctypes.c_int * b)(*n) for n in (q_lens, kv_lens))
        ws_bytes = _lib.on_device(dev, _lib.load().vomni_attention_bwd_workspace_bytes, b, sq, skv, hq, hkv, _HEAD_DIM, q_lens, kv_lens)
    ws = _lib.workspace(ws_bytes, q.device)
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), b, sq, skv, hq, hkv, _HEAD_DIM, strides, q_lens, kv_lens,
            scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes)
    if grad_lse is None:
        _lib.launch(dev, "vomni_attention_bwd", grad_o.data_ptr(), *args)
    else:
        _lib.launch(dev, "vomni_attention_bwd_lse", grad_o.data_ptr(), grad_lse.data_ptr(), *args)
    return dq, dk, dv


def wan_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None, *, q_lens=None,
                  kv_lens=None) -> torch.Tensor:
    """Differentiable attention ``[b, hq, s_q, 128]`` of one device's ``q [b, s_q, hq, 128]``, ``k, v [b, s_kv, hkv, 128]``;
    the arguments are those of :func:`attention_fwd`, the gradients those of :func:`attention_bwd`."""
    return attention_fwd(q, k, v, softmax_scale, q_lens=q_lens, kv_lens=kv_lens)[0]
