"""The C entries of the norms around a block with outputs in place of inputs, as their contract allows: the bits of the call with
outputs of their own (B200 only). Widths and rows reach each kernel: rows that are part of a warp (256 columns and less), one, two and four
rows at a time, and the backward pass of many rows."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(1, 5, 64), (2, 700, 128), (1, 3000, 256), (1, 7, 520), (2, 333, 1536), (1, 2500, 1536), (1, 1300, 5120), (1, 1200, 5000),
          (1, 900, 6000), (2, 40, 8192)]
EPS, RMS, LAYER = 1e-6, 1, 0


@pytest.fixture(scope="module")
def lib(pkg):
    from importlib import import_module

    return import_module("vllm-omni-neuron_b200._lib")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _make(dev, b, s, h, n):
    g = torch.Generator().manual_seed(s + h)
    rows = [torch.randn(b * s, h, generator=g).to(torch.bfloat16).to(dev) for _ in range(n)]
    return rows, [torch.randn(b, h, generator=g).to(dev) for _ in range(3)], torch.randn(h, generator=g).to(dev)


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("b,s,h", SHAPES)
def test_forward(lib, dev, b, s, h):
    (x, res), (gate, mul, add), w = _make(dev, b, s, h, 2)

    def run(x, res, res_out, out):
        lib.call("vomni_sandwich_norm", _ptr(x), _ptr(res), None if x is None else _ptr(gate), None if x is None else _ptr(w), _ptr(mul),
                 _ptr(add), b * s, h, s, 7, EPS, RMS, LAYER, _ptr(res_out), _ptr(out), _stream())
        torch.cuda.synchronize()
        return res_out, out

    want = run(x, res, torch.empty_like(x), torch.empty_like(x))
    first = run(None, res, None, torch.empty_like(x))[1]
    for of_res, of_out in (("x", None), ("res", None), (None, "x"), (None, "res"), ("x", "res"), ("res", "x")):
        t = {"x": x.clone(), "res": res.clone(), None: torch.empty_like(x)}
        more = torch.empty_like(x)
        got = run(t["x"], t["res"], t[of_res] if of_res else more, t[of_out])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (of_res, of_out)
    again = res.clone()
    assert torch.equal(run(None, again, None, again)[1], first)


@pytest.mark.parametrize("b,s,h", SHAPES)
@pytest.mark.parametrize("norms", [(RMS, LAYER), (LAYER, RMS)])
def test_backward(lib, dev, b, s, h, norms):
    (gr, go, x, res), (gate, mul, _), w = _make(dev, b, s, h, 4)
    ws = lib.workspace(lib.workspace_bytes(dev.index, "vomni_sandwich_norm", b * s, h, s), dev)

    def run(gr, go, x, dx, dres):
        sums = [torch.empty(b, h, device=dev), torch.empty(h, device=dev), torch.empty(b, h, device=dev), torch.empty(b, h, device=dev)]
        if x is None:
            sums[0] = sums[1] = None
        lib.call("vomni_sandwich_norm_bwd", _ptr(gr), _ptr(go), _ptr(x), _ptr(res), None if x is None else _ptr(gate),
                 None if x is None else _ptr(w), _ptr(mul), b * s, h, s, 7, EPS, *norms, _ptr(dx), _ptr(dres), *map(_ptr, sums),
                 _ptr(ws), ws.numel(), _stream())
        torch.cuda.synchronize()
        return [t for t in (dx, dres, *sums) if t is not None]

    same = lambda a, c: len(a) == len(c) and all(torch.equal(m, n) for m, n in zip(a, c))
    new = lambda: torch.empty_like(x)
    for has in ((True, True), (True, False), (False, True)):
        args = [t if keep else None for t, keep in zip((gr, go), has)]
        want, first = run(*args, x, new(), new()), run(*args, None, None, new())
        for i, j in ((0, None), (1, None), (None, 0), (None, 1), (0, 1), (1, 0)):  # gradient in whose place dx, dresidual go
            a = [None if t is None else t.clone() for t in args]
            if any(n is not None and a[n] is None for n in (i, j)):
                continue
            assert same(run(*a, x, new() if i is None else a[i], new() if j is None else a[j]), want), (has, i, j)
            if i is None:
                a = [None if t is None else t.clone() for t in args]
                assert same(run(*a, None, None, a[j]), first), (has, j)


def test_residual_out_without_a_branch_is_refused(lib, dev):
    (x, res), _, _ = _make(dev, 1, 8, 64, 2)
    kept = x.clone()
    with pytest.raises(lib.VomniError) as e:
        lib.call("vomni_sandwich_norm", None, _ptr(res), None, None, None, None, 8, 64, 8, 0, EPS, RMS, LAYER, _ptr(x), _ptr(kept),
                 _stream())
    assert e.value.code == 1
