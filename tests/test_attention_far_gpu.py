"""Attention forward and backward of rows whose scores lie far below the Cauchy-Schwarz bound scale |q| max |k|, or whose bound is too
large for its own rounding (B200 only), against the definition in 64 bits.

Tolerances. A score is a sum of 128 products in fp32: 128 * 2^-24 of the sum of their magnitudes, times scale. The exponential's argument
and lse are formed from numbers of the bound's size with a few roundings (2^-21 of the bound). Both move P relatively (E below). P is
rounded to bf16 (2^-8) for the products; o is divided by a sum of such P (2^-8 more) and rounded (2^-8); lse is the log of a sum of P, rounded to
bf16 or not (2^-8). The gradients' own bounds are those of test_attention_bwd_gpu, with P off by 2^-8 and twice E (scores and lse)."""

import math

import pytest
import torch

from test_attention_bwd_gpu import ACC, HALF, _check, _forward, _grads, _scores

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _rows(lse, sq):
    return lse.transpose(2, 3).flatten(2)[..., :sq]


def _compare(pkg, q, k, v, go, scale=SCALE, lens=None, kv_lens=None):
    hq, hkv, sq = q.shape[2], k.shape[2], q.shape[1]
    n = hq // hkv
    o, lse = pkg.attention_fwd(q, k, v, scale, q_lens=lens, kv_lens=kv_lens)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    again = pkg.wan_attention(*leaves, scale, q_lens=lens, kv_lens=kv_lens)
    assert torch.equal(o, again.detach())
    grads = torch.autograd.grad(again, leaves, go)
    ro, rl = _forward(q, k, v, scale, lens, kv_lens)
    s, keep = _scores(q, k, scale, lens, kv_lens)
    there = ~rl.isinf()
    p = torch.where(keep & there[..., None], torch.exp(s - torch.where(there, rl, 0.0)[..., None]), 0.0)
    kk, vv = (t.double().transpose(1, 2).repeat_interleave(n, 1).abs() for t in (k, v))
    qa = q.double().transpose(1, 2).abs()
    bound = scale * qa.square().sum(-1).sqrt() * kk.square().sum(-1).sqrt().amax(-1, keepdim=True)
    e = (ACC * scale * (qa @ kk.transpose(2, 3))).amax(-1) + 2.0**-21 * bound  # [b, h, sq]
    assert e.max() < 0.25, "the bounds say nothing"
    assert torch.equal(_rows(lse, sq).isinf(), ~there)
    off = torch.where(there, (_rows(lse, sq).double() - rl).abs(), 0.0)
    assert (off <= 2 * e + HALF + k.shape[1] * 2.0**-24).all(), f"lse: {(off - 2 * e).max():.4g}"
    mag = p @ vv
    o_off = (4 * e[..., None] + 2 * HALF + k.shape[1] * 2.0**-24) * mag + HALF * ro.abs() + 1e-30
    assert ((o.double() - ro).abs() <= o_off).all(), f"o: {((o.double() - ro).abs() / o_off).max():.3f} of the bound"
    want, room = _grads(q, k, v, ro, rl, go, scale, lens, kv_lens, e_p=HALF + 4 * e[..., None])
    more = p * (go.double().abs() * o_off).sum(-1, keepdim=True)  # o moves delta
    fold = lambda t: t.unflatten(1, (hkv, n)).sum(2).transpose(1, 2)
    _check(grads, want, (room[0] + (scale * more @ kk).transpose(1, 2), room[1] + fold(scale * more.transpose(2, 3) @ qa), room[2]))
    return o, lse


def _normal(dev, b, sq, skv, hq, hkv, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)
    t = (mk(b, sq, hq, 128) * size, mk(b, skv, hkv, 128) * size, mk(b, skv, hkv, 128) + 0.25, mk(b, hq, sq, 128) * 0.05)
    return [x.to(torch.bfloat16).to(dev) for x in t]


@pytest.mark.parametrize("bound", [10.0, 30.0, 44.0, 60.0, 250.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_one_key(pkg, dev, bound, sign):
    """q = a k or -a k: the one score is +-bound, the probability 1, o = v and dq = dk = 0."""
    g = torch.Generator().manual_seed(int(bound))
    k = torch.randn(1, 1, 2, 128, generator=g).to(torch.bfloat16)
    a = bound / (SCALE * k.double().square().sum(-1, keepdim=True))
    q = (sign * a * k.double()).expand(1, 70, 2, 128).to(torch.bfloat16)
    v = torch.randn(1, 1, 2, 128, generator=g).to(torch.bfloat16)
    go = torch.randn(1, 2, 70, 128, generator=g).to(torch.bfloat16)
    q, k, v, go = (t.to(dev) for t in (q, k, v, go))
    o, _ = _compare(pkg, q, k, v, go)
    assert torch.equal(o, v.transpose(1, 2).expand(1, 2, 70, 128))


@pytest.mark.parametrize("skv", [2, 65, 700, 5000])
@pytest.mark.parametrize("gap", [40.0, 50.0, 60.0, 80.0, 86.0, 88.0, 100.0, 400.0])
def test_all_keys_far_below_the_bound(pkg, dev, skv, gap):
    """Ordinary scores, and one key of a large norm across q that sets the bound `gap` above them; half the rows have small q, whose
    bound is near, in the same tiles."""
    q, k, v, go = _normal(dev, 1, 150, skv, 2, 2, int(gap) + skv)
    q[..., 64:] = 0
    q[:, ::2] *= 0.25
    k[:, skv // 2] = 0
    norm = q[:, 1::2].double().square().sum(-1).sqrt().mean()
    k[:, skv // 2, :, 64:] = (gap / (SCALE * norm * 8.0)).to(torch.bfloat16)  # 64 equal values: norm 8 times one
    _compare(pkg, q, k, v, go)


@pytest.mark.parametrize("size", [2.0, 2.5, 3.0, 6.0, 12.0])
def test_large_norms(pkg, dev, size):
    _compare(pkg, *_normal(dev, 2, 300, 333, 2, 2, 3, size))


@pytest.mark.parametrize("b,sq,skv,hq,hkv,lens,kv_lens", [
    (3, 300, 400, 4, 2, [300, 77, 0], [400, 1, 131]),
    (2, 65, 64, 6, 1, None, None),
    (2, 1, 130, 3, 3, None, [130, 0]),
    (1, 1000, 17, 5, 5, None, None),
])
def test_lengths_and_shared_heads(pkg, dev, b, sq, skv, hq, hkv, lens, kv_lens):
    _compare(pkg, *_normal(dev, b, sq, skv, hq, hkv, 4, 4.0), lens=lens, kv_lens=kv_lens)


def test_scales(pkg, dev):
    _compare(pkg, *_normal(dev, 1, 130, 200, 2, 2, 5, 2.0), scale=0.5)
    _compare(pkg, *_normal(dev, 1, 130, 200, 2, 2, 6, 8.0), scale=0.02)


def test_a_bound_beyond_fp32(pkg, dev):
    """Norms whose squares' product overflows fp32: the bound is infinite, the scores are not."""
    q, k, v, go = _normal(dev, 1, 70, 90, 1, 1, 7)
    with pytest.raises(ValueError):  # scales below 1e-20
        pkg.attention_fwd(q * 2.0**60, k * 2.0**60, v, 2.0**-120 / 8)
    q, k, scale = q * 2.0**30, k * 2.0**33, 2.0**-66
    o, lse = pkg.attention_fwd(q, k, v, scale)
    ro, rl = _forward(q, k, v, scale)
    s, _ = _scores(q, k, scale, None, None)
    e = (ACC * scale * (q.double().transpose(1, 2).abs() @ k.double().transpose(1, 2).abs().transpose(2, 3))).amax(-1) + 2.0**-20
    p = torch.exp(s - rl[..., None])
    assert ((_rows(lse, 70).double() - rl).abs() <= 2 * e + HALF).all()
    assert ((o.double() - ro).abs() <= (4 * e[..., None] + 2 * HALF) * (p @ v.double().transpose(1, 2).abs()) + HALF * ro.abs()).all()


def test_near_rows_keep_their_bits(pkg, dev):
    """Rows that the bound fits are what ring_attention_const_max_fwd gives, also in tiles with rows that it does not."""
    q, k, v, _ = _normal(dev, 2, 200, 200, 2, 2, 8)
    q[:, 3::7] *= 40.0
    o, lse = pkg.attention_fwd(q, k, v)
    ro, rl = pkg.ring_attention_const_max_fwd(q, k, v, training=True)
    near = torch.ones(200, dtype=torch.bool, device=dev)
    near[3::7] = False
    assert torch.equal(o[:, :, near], ro[:, :, near]) and torch.equal(_rows(lse, 200)[..., near], _rows(rl, 200)[..., near])
    assert not torch.equal(o, ro)


def test_not_a_number_stays_in_its_row(pkg, dev):
    q, k, v, _ = _normal(dev, 1, 140, 90, 1, 1, 9, 4.0)
    o, lse = pkg.attention_fwd(q, k, v)
    q[:, 77, 0, 5] = math.nan
    o2, lse2 = pkg.attention_fwd(q, k, v)
    assert o2[0, 0, 77].isnan().all() and _rows(lse2, 140)[0, 0, 77].isnan()
    rest = torch.arange(140, device=dev) != 77
    assert torch.equal(o[:, :, rest], o2[:, :, rest]) and torch.equal(_rows(lse, 140)[..., rest], _rows(lse2, 140)[..., rest])


def test_views_streams_and_graphs(pkg, dev):
    """Column slices of a fused projection, another stream, and a captured call: the same bits."""
    q, k, v, _ = _normal(dev, 2, 193, 193, 3, 3, 10, 4.0)
    o, lse = pkg.attention_fwd(q, k, v)
    fused = torch.cat([t.flatten(2) for t in (q, k, v)], dim=-1)
    views = [t.unflatten(2, (3, 128)) for t in fused.chunk(3, dim=-1)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = pkg.attention_fwd(*views)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = pkg.attention_fwd(*views)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a in (other, kept):
        assert torch.equal(a[0], o) and torch.equal(a[1], lse)


def test_far_offsets(pkg, dev):
    """Element offsets past 2^31."""
    q, k, v, _ = _normal(dev, 1, 300, 300, 1, 1, 11, 4.0)
    o, lse = pkg.attention_fwd(q, k, v)
    far = torch.empty_strided((1, 300, 1, 128), (300 << 23, 1 << 23, 128, 1), dtype=torch.bfloat16, device=dev)
    far.copy_(q)
    a = pkg.attention_fwd(far, k, v)
    assert torch.equal(a[0], o) and torch.equal(a[1], lse)
