"""A loss on the log-sum-exp alone, through the training forward, against the definition in 64 bits (B200 only): dS = P grad_lse.

dS is rounded to bf16 (2^-8), P is off by its lse's error (2^-8, the rounding of the probabilities that lse sums) and by the exponential's
(2^-18); the products are sums in fp32 (2^-24 a term), the results rounded once (2^-8). Without grad_o the rest of dS is exactly 0."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0**-8
SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("b,sq,skv,hq,hkv,kv_lens", [(1, 130, 70, 2, 2, None), (2, 300, 513, 4, 2, None), (2, 77, 200, 2, 1, [131, 1])])
def test_against_definition(pkg, dev, b, sq, skv, hq, hkv, kv_lens):
    g = torch.Generator().manual_seed(sq)
    mk = lambda *s: torch.randn(*s, generator=g)
    q, k, v = (t.to(torch.bfloat16).to(dev).requires_grad_(True) for t in (mk(b, sq, hq, 128), mk(b, skv, hkv, 128), mk(b, skv, hkv, 128)))
    gl = mk(b, hq, sq).to(dev)
    rows = lambda lse: lse.transpose(2, 3).flatten(2)[..., :sq]
    got = torch.autograd.grad((rows(pkg.attention_fwd(q, k, v, kv_lens=kv_lens)[1]) * gl).sum(), (q, k, v))
    n = hq // hkv
    qd, kd = q.detach().double().transpose(1, 2), k.detach().double().transpose(1, 2).repeat_interleave(n, 1)
    s = SCALE * qd @ kd.transpose(2, 3)
    if kv_lens:
        s = s.masked_fill(~(torch.arange(skv, device=dev)[None] < torch.tensor(kv_lens, device=dev)[:, None])[:, None, None], -math.inf)
    ds = torch.softmax(s, -1) * gl.double()[..., None]
    fold = lambda t: t.unflatten(1, (hkv, n)).sum(2).transpose(1, 2)
    rel = 2 * HALF + 2.0**-18 + max(sq * n, skv) * 2.0**-24
    for x, want, mag in ((got[0], (SCALE * ds @ kd).transpose(1, 2), (SCALE * ds.abs() @ kd.abs()).transpose(1, 2)),
                         (got[1], fold(SCALE * ds.transpose(2, 3) @ qd), fold(SCALE * ds.abs().transpose(2, 3) @ qd.abs()))):
        assert ((x.double() - want).abs() <= rel * mag + HALF * want.abs() + 1e-30).all()
    assert not got[2].any()
