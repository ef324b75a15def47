"""Gradients of the norms around a block over many rows (several groups of rows a CTA, the last one short), against the definition
in 64 bits with the tolerances of the short ones (B200 only)."""

import itertools

import pytest
import torch
from test_sandwich_gpu import KINDS, _check_backward, _check_forward, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("post,norm", list(itertools.product(KINDS, KINDS)))
@pytest.mark.parametrize("lead,h", [((2, 3333), 520), ((1, 3001), 2048), ((1501,), 5120)])
def test_kinds(pkg, dev, lead, h, post, norm):
    st = _make(dev, lead, h, h + len(post))
    _check_backward(pkg, st, _check_forward(pkg, st, post, norm), post, norm)


@pytest.mark.parametrize("h", [264, 640, 1000, 4104, 5112, 6000, 8192])
def test_sizes(pkg, dev, h):
    st = _make(dev, (1, 2011), h, h, per=("gate",))
    _check_backward(pkg, st, _check_forward(pkg, st, "layer_norm", "layer_norm"), "layer_norm", "layer_norm")


@pytest.mark.parametrize("lead", [(1, 1), (7,), (2, 33), (3, 5001)])
@pytest.mark.parametrize("h", [8, 64, 72, 128, 200, 256])
def test_short_rows(pkg, dev, lead, h):
    """Several rows a warp, or one."""
    for post, norm in (("rms_norm", "layer_norm"), ("layer_norm", "none")):
        st = _make(dev, lead, h, h + len(post), per=("mul", "add"))
        _check_backward(pkg, st, _check_forward(pkg, st, post, norm), post, norm)


@pytest.mark.parametrize("per", [("gate", "mul", "add"), ("gate",), ("mul",), ("add",)])
@pytest.mark.parametrize("lead,h", [((8, 3), 264), ((9, 2), 128), ((64, 1), 1536), ((65, 7), 72), ((333, 1), 2048), ((1000, 2), 264)])
def test_many_modulation_rows(pkg, dev, lead, h, per):
    """Up to one modulation row per token; the shared vectors' gradients are sums over all of them."""
    st = _make(dev, lead, h, h + lead[0], per=per)
    _check_backward(pkg, st, _check_forward(pkg, st, "rms_norm", "layer_norm"), "rms_norm", "layer_norm")


@pytest.mark.parametrize("missing", ["grad_r", "grad_out", "x"])
def test_parts_of_a_call(pkg, dev, missing):
    st = _make(dev, (3, 1001), 1536, 7, branch=missing != "x")
    r = _check_forward(pkg, st, "rms_norm", "layer_norm")
    if missing != "x":
        st[missing] = None
    _check_backward(pkg, st, r, "rms_norm", "layer_norm")


def test_same_bits_on_every_stream(pkg, dev):
    st = _make(dev, (2, 3333), 1536, 9)
    call = lambda: pkg.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], st["residual"], st["gate"], st["mul"], st["add"], eps=1e-6,
                                         post_weight=st["post_weight"])
    want = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))
