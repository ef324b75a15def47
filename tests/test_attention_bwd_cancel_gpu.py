"""Gradients that vanish (B200 only): where every key of a row has one and the same value vector v, O = v whatever the
probabilities are, dP = dO v = delta for every key, and dQ = dK = 0 exactly. A row with one key is the smallest such row.
dP and delta are sums of the same 128 products, so no rounding may be left between them: the bound is 0. dV is P^T dO, with P rounded
to bf16 (2^-8, and 2^-18 of the exponential), summed in fp32 (2^-24 a term) and rounded once (2^-8)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _case(dev, b, sq, skv, hq, hkv, q_lens, kv_lens, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    q, k, go = mk(b, sq, hq, 128), mk(b, skv, hkv, 128), mk(b, hq, sq, 128)
    v = mk(b, 1, hkv, 128).repeat(1, skv, 1, 1)  # of all keys of a head
    n = hq // hkv
    s = SCALE * q.double().transpose(1, 2) @ k.double().transpose(1, 2).repeat_interleave(n, 1).transpose(2, 3)
    ql, kl = (torch.tensor(x or [m] * b, device=dev) for x, m in ((q_lens, sq), (kv_lens, skv)))
    rows = (torch.arange(sq, device=dev)[None] < ql[:, None])[:, None, :, None]
    keep = rows & (torch.arange(skv, device=dev)[None] < kl[:, None])[:, None, None, :]
    lse = torch.logsumexp(s.masked_fill(~keep, -math.inf), -1)
    there = ~lse.isinf()[..., None]
    p = torch.where(keep, torch.exp(s - torch.where(there[..., 0], lse, 0.0)[..., None]), 0.0)
    o = torch.where(there, v[:, :1].transpose(1, 2).repeat_interleave(n, 1).expand(b, hq, sq, 128), 0.0).to(torch.bfloat16)
    groups = -(-sq // 128)
    full = torch.zeros(b, hq, groups * 128, dtype=torch.float32, device=dev)
    full[:, :, :sq] = lse.float()
    return q, k, v, go, o, full.reshape(b, hq, groups, 128).transpose(2, 3).contiguous(), p


CASES = [
    (1, 1, 1, 1, 1, None, None),
    (1, 77, 1, 4, 4, None, None),
    (2, 300, 1, 8, 4, None, None),
    (1, 5000, 1, 8, 8, None, None),
    (2, 300, 300, 4, 2, [300, 200], [1, 1]),
    (3, 140, 20, 2, 1, [140, 1, 0], [1, 0, 1]),
    (1, 1, 1, 40, 40, None, None),
    (2, 1, 300, 3, 1, None, None),
    (1, 400, 700, 2, 2, None, None),
    (2, 513, 257, 3, 1, [513, 130], [257, 129]),
    (1, 130, 5000, 1, 1, None, None),
]


@pytest.mark.parametrize("case", CASES)
def test_exactly_zero(pkg, dev, case):
    b, sq, skv, hq, hkv, q_lens, kv_lens = case
    q, k, v, go, o, lse, p = _case(dev, *case, seed=sq + 7 * skv)
    dq, dk, dv = pkg.attention_bwd(go, q, k, v, o, lse, SCALE, q_lens=q_lens, kv_lens=kv_lens)
    assert not dq.any() and not dk.any()
    fold = lambda t: t.unflatten(1, (hkv, hq // hkv)).sum(2).transpose(1, 2)
    want, mag = fold(p.transpose(2, 3) @ go.double()), fold(p.transpose(2, 3) @ go.double().abs())
    bound = (2.0**-8 + 2.0**-18 + sq * hq // hkv * 2.0**-24) * mag + 2.0**-8 * want.abs() + 1e-30
    assert ((dv.double() - want).abs() <= bound).all()
    again = pkg.attention_bwd(go, q, k, v, o, lse, SCALE, q_lens=q_lens, kv_lens=kv_lens)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))


@pytest.mark.parametrize("skv", [1, 200])
def test_what_the_lse_s_gradient_adds_is_alone(pkg, dev, skv):
    """With grad_lse = c, dS = P c: the rest is exactly 0, so dQ = scale c P K and dK = scale P^T c Q."""
    q, k, v, go, o, lse, p = _case(dev, 1, 150, skv, 2, 2, None, None, seed=3)
    c = torch.randn(1, 2, 150, generator=torch.Generator().manual_seed(4)).to(dev)
    full = torch.zeros(1, 2, 256, device=dev)
    full[:, :, :150] = c
    got = pkg.attention_bwd(go, q, k, v, o, lse, SCALE, grad_lse=full.reshape(1, 2, 2, 128).transpose(2, 3).contiguous())
    ds = p * c.double()[..., None]
    # dP - (delta - c) in fp32: the difference of two values of |delta| + |c| at most, each off by half a step of fp32 (2^-24), and by a
    # step (2^-23) where the tensor cores truncate
    delta = (go.double() * o.double()).sum(-1).abs()
    off = (p * ((2.0**-8 + 2.0**-18) * c.double().abs() + 2.0**-22 * (delta + c.double().abs()))[..., None]) * (1 + 200 * 2.0**-24)
    kd, qd = k.double().transpose(1, 2), q.double().transpose(1, 2)
    for x, want, e in ((got[0], SCALE * ds @ kd, SCALE * off @ kd.abs()), (got[1], SCALE * ds.transpose(2, 3) @ qd, SCALE * off.transpose(2, 3) @ qd.abs())):
        assert ((x.double().transpose(1, 2) - want).abs() <= e + 2.0**-8 * want.abs() + 200 * 2.0**-24 * want.abs() + 1e-30).all()
