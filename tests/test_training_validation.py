"""Refusals of the training operators, on the CPU: every check runs before any device call."""

import ctypes

import pytest
import torch


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.fixture(scope="module")
def lib(pkg):
    from importlib import import_module

    return import_module("vllm-omni-neuron_b200._lib").load()


def test_attention(pkg):
    q, o, lse = _bf(2, 16, 4, 128), _bf(2, 4, 16, 128), torch.zeros(2, 4, 128, 1)
    bwd = lambda **kw: pkg.attention_bwd(*(kw.get(n, d) for n, d in
                                           (("go", o), ("q", q), ("k", q), ("v", q), ("o", o), ("lse", lse))),
                                         q_lens=kw.get("q_lens"), kv_lens=kw.get("kv_lens"))
    with pytest.raises(RuntimeError):  # no CPU path
        bwd()
    with pytest.raises(TypeError):
        bwd(q=q.float())
    with pytest.raises(TypeError):
        bwd(go=o.half())
    with pytest.raises(ValueError):  # head dim
        bwd(q=_bf(2, 16, 4, 64), k=_bf(2, 16, 4, 64), v=_bf(2, 16, 4, 64))
    with pytest.raises(ValueError):  # 4 query heads over 3 key heads
        bwd(k=_bf(2, 16, 3, 128), v=_bf(2, 16, 3, 128))
    with pytest.raises(ValueError):
        bwd(v=_bf(2, 17, 4, 128))
    with pytest.raises(ValueError):  # token-major output
        bwd(o=_bf(2, 16, 4, 128))
    with pytest.raises(ValueError):
        bwd(lse=torch.zeros(2, 4, 16))
    with pytest.raises(ValueError):
        bwd(q_lens=[16])
    with pytest.raises(ValueError):
        bwd(kv_lens=[3, 17])
    with pytest.raises(ValueError):
        bwd(kv_lens=[-1, 3])
    with pytest.raises(TypeError):  # a device tensor of lengths would need a synchronisation
        bwd(kv_lens=torch.tensor([3, 4]))
    for bad in (0.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            pkg.attention_bwd(o, q, q, q, o, lse, bad)
        with pytest.raises(ValueError):
            pkg.attention_fwd(q, q, q, bad)
    with pytest.raises(ValueError):  # the softmax bound is a norm: positive scales only
        pkg.wan_attention(q, q, q, -0.1)
    with pytest.raises(RuntimeError):
        pkg.attention_fwd(q, q, q)
    with pytest.raises(RuntimeError):
        pkg.wan_attention(q, q, q, q_lens=[1, 2])


def test_rotary(pkg):
    q, pos = _bf(2, 8, 4, 128), torch.zeros(8, 3, dtype=torch.int32)
    axes = (44, 42, 42)
    with pytest.raises(RuntimeError):
        pkg.rotary_axes(q, q, pos, axes)
    with pytest.raises(TypeError):
        pkg.rotary_axes(q.double(), None, pos, axes)
    with pytest.raises(TypeError):
        pkg.rotary_axes(q, q.float(), pos, axes)
    with pytest.raises(TypeError):
        pkg.rotary_axes(q, q, pos.double(), axes)
    with pytest.raises(ValueError):
        pkg.rotary_axes(q, q[:, :4], pos, axes)
    with pytest.raises(ValueError):
        pkg.rotary_axes(q[0], None, pos, axes)
    for bad in ((44, 42), (43, 43, 42), (128, 0, 0), (16, 16, 32, 32, 32), ()):
        with pytest.raises(ValueError):
            pkg.rotary_axes(q, q, pos, bad)
    for bad in (pos[:4], pos[:, :2], pos[None].expand(3, -1, -1)):
        with pytest.raises(ValueError):
            pkg.rotary_axes(q, q, bad, axes)
    with pytest.raises(ValueError):
        pkg.rotary_axes(q, q, pos, axes, pairing="neox")
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            pkg.rotary_axes(q, q, pos, axes, theta=theta)
    with pytest.raises(ValueError):
        pkg.rotary_axes(_bf(1, 8, 1, 24), None, pos, (8, 8, 8))


def test_sandwich(pkg):
    x, g = _bf(2, 8, 64), torch.zeros(2, 1, 64)
    with pytest.raises(RuntimeError):
        pkg.sandwich_norm(x, x, g, g, g, eps=1e-6)
    with pytest.raises(TypeError):
        pkg.sandwich_norm(x, x, g.double(), eps=1e-6)
    with pytest.raises(ValueError):
        pkg.sandwich_norm(x, x, torch.zeros(3, 1, 64), eps=1e-6)
    with pytest.raises(ValueError):
        pkg.sandwich_norm(x, x, torch.zeros(32), eps=1e-6)
    with pytest.raises(ValueError):
        pkg.sandwich_norm(x, x, post_weight=g, eps=1e-6)
    with pytest.raises(ValueError):
        pkg.sandwich_norm(x, x, eps=1e-6, post_norm="batch_norm")
    with pytest.raises(ValueError):
        pkg.sandwich_norm(x, x, eps=1e-6, norm_type="batch_norm")
    with pytest.raises(ValueError):  # gate scales a branch that is not there
        pkg.sandwich_norm(None, x, g, eps=1e-6)
    for bad in (_bf(2, 8, 12), _bf(1, 8200), _bf(64)):
        with pytest.raises(ValueError):
            pkg.sandwich_norm(bad, bad, eps=1e-6)
    for eps in (0.0, -1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            pkg.sandwich_norm(x, x, eps=eps)
    many = _bf(70000, 1, 8)
    with pytest.raises(ValueError):
        pkg.sandwich_norm(many, many, torch.zeros(70000, 1, 8), eps=1e-6)
    with pytest.raises(ValueError):
        pkg.sandwich_norm_bwd(None, None, x, x, eps=1e-6)


def test_c_entries(lib):
    """Status codes of the C ABI, with pointers that are never read."""
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)
    ok = (ctypes.c_longlong * 15)(*([512, 128, 512 * 16] * 5))

    def bwd(b=2, sq=16, skv=16, hq=4, hkv=4, d=128, strides=ok, ql=None, kl=None, ws=1 << 40, dq=p, q=p, scale=0.1):
        ints = lambda v: (ctypes.c_int * len(v))(*v) if v else None
        return lib.vomni_attention_bwd(p, q, p, p, p, p, b, sq, skv, hq, hkv, d, strides, ints(ql), ints(kl), scale, dq, p, p, p, ws,
                                       None)

    assert bwd(dq=None) == 1 and bwd(scale=0.0) == 1 and bwd(scale=float("nan")) == 1 and bwd(scale=1e30) == 1
    assert bwd(d=64) == 2 and bwd(hkv=3) == 2 and bwd(sq=0) == 2 and bwd(b=5000) == 2
    assert bwd(ql=[17, 1]) == 2 and bwd(kl=[-1, 1]) == 2
    assert bwd(q=odd) == 3
    assert bwd(strides=(ctypes.c_longlong * 15)(*([513, 128, 512 * 16] * 5))) == 3
    assert bwd(strides=(ctypes.c_longlong * 15)(*([0, 128, 512 * 16] * 5))) == 3
    assert bwd(ws=64) == 8
    assert lib.vomni_attention_bwd_workspace_bytes(1, 16, 16, 4, 3, 128, None, None) == 0
    assert lib.vomni_attention_bwd_workspace_bytes(2, 200, 16, 4, 4, 128, None, None) >= 2 * 2 * 4 * 256 * 4

    axes = (ctypes.c_int * 3)(44, 42, 42)

    def rotary(qh=4, kh=4, b=2, s=8, d=128, n=3, a=axes, theta=1e4, pos_type=0, pairing=0, dtype=0, q=p, row=512):
        return lib.vomni_rotary_axes(q, p, qh, row, 4096, p, p, kh, 512, 4096, b, s, d, p, pos_type, 0, n, a, theta, pairing, 0, dtype,
                                     None)

    assert rotary(q=None) == 1 and rotary(theta=0.0) == 1 and rotary(theta=float("nan")) == 1
    assert rotary(pos_type=3) == 1 and rotary(pairing=2) == 1 and rotary(dtype=3) == 1
    assert rotary(d=120) == 2 and rotary(n=2) == 2 and rotary(n=5) == 2 and rotary(s=0) == 2 and rotary(row=256) == 2
    assert rotary(a=(ctypes.c_int * 3)(45, 41, 42)) == 2 and rotary(a=(ctypes.c_int * 3)(64, 64, 64)) == 2
    assert rotary(q=odd) == 3 and rotary(row=513) == 3

    def norm(x=p, res=p, gate=None, w=None, rows=8, h=64, per=8, bits=0, post=1, kind=0, r=p, out=p):
        return lib.vomni_sandwich_norm(x, res, gate, w, None, None, rows, h, per, bits, 1e-6, post, kind, r, out, None)

    assert norm(res=None) == 1 and norm(r=None) == 1 and norm(bits=8) == 1 and norm(post=3) == 1 and norm(kind=-1) == 1
    assert norm(x=None, gate=p) == 1
    assert norm(rows=70000, per=1) == 2
    assert norm(h=12) == 2 and norm(h=8200) == 2 and norm(rows=0) == 2 and norm(per=3) == 2
    assert norm(x=odd) == 3

    def grad(gr=p, go=p, x=p, res=p, gate=None, rows=8, h=64, per=8, dx=p, dres=p, dgate=None, ws=1 << 40):
        return lib.vomni_sandwich_norm_bwd(gr, go, x, res, gate, None, None, rows, h, per, 0, 1e-6, 1, 0, dx, dres, dgate, None, None,
                                           None, p, ws, None)

    assert grad(gr=None, go=None) == 1 and grad(dx=None) == 1 and grad(dres=None) == 1 and grad(res=None) == 1
    assert grad(x=None) == 1 and grad(x=None, dx=None, dgate=p) == 1
    assert grad(rows=0) == 2 and grad(per=3) == 2 and grad(rows=70000, per=1) == 2
    assert grad(go=odd) == 3 and grad(ws=64) == 8
    assert lib.vomni_sandwich_norm_workspace_bytes(8, 12, 8) == 0
