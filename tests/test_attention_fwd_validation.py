"""Refusals of the C entry of the training forward, on the CPU: every check runs before any device call."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib(pkg):
    from importlib import import_module

    return import_module("vllm-omni-neuron_b200._lib").load()


def test_attention_fwd(lib):
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)

    def fwd(q=p, k=p, v=p, o=p, lse=p, b=1, sq=16, skv=16, h=4, d=128, qs=0, ks=0, scale=0.1, ws=p, n=1 << 40):
        return lib.vomni_attention_fwd(q, k, v, o, lse, b, sq, skv, h, d, qs, ks, scale, ws, n, None)

    assert fwd(lse=None) == 1 and fwd(q=None) == 1 and fwd(ws=None) == 1 and fwd(o=None) == 1 and fwd(v=None) == 1
    for scale in (0.0, -0.1, 1e-30, 1e30, float("nan"), float("inf")):
        assert fwd(scale=scale) == 1
    assert fwd(d=64) == 2 and fwd(sq=0) == 2 and fwd(skv=0) == 2 and fwd(h=0) == 2 and fwd(qs=8) == 2
    assert fwd(q=odd) == 3 and fwd(k=odd) == 3 and fwd(v=odd) == 3 and fwd(o=odd) == 3 and fwd(qs=513) == 3
    assert fwd(n=64) == 8
