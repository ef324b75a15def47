"""The attention's gradients where its log-sum-exp is used too, against the definition in 64 bits (B200 only).

d lse_i / d s_ij = P_ij, so a gradient of lse enters dS beside -delta. Tolerances are those of the gradients without it (P and dS
rounded to bf16, 2^-8 relative each; the results once, 2^-8; sums in fp32), with |grad_lse| among the magnitudes that make dS."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0**-8
SCALE = 1 / math.sqrt(128)


def _make(dev, b, sq, skv, hq, hkv, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)
    q, k, v, go = mk(b, sq, hq, 128), mk(b, skv, hkv, 128), mk(b, skv, hkv, 128) + 0.25, mk(b, hq, sq, 128) * 0.05
    return [t.to(torch.bfloat16).to(dev) for t in (q, k, v, go)] + [(mk(b, hq, sq)).to(dev)]


def _layout(rows, fill=0.0):
    b, h, s = rows.shape
    g = -(-s // 128)
    full = torch.full((b, h, g * 128), fill, dtype=torch.float32, device=rows.device)
    full[:, :, :s] = rows.float()
    return full.reshape(b, h, g, 128).transpose(2, 3).contiguous()


def _definition(q, k, v, kv_lens=None):
    """(o, lse rows) of rows that have keys, in the inputs' type; 0 and -inf where a batch element has none."""
    n = q.shape[2] // k.shape[2]
    k, v = (t.transpose(1, 2).repeat_interleave(n, dim=1) for t in (k, v))
    s = SCALE * q.transpose(1, 2) @ k.transpose(2, 3)
    if kv_lens:
        keep = torch.arange(s.shape[-1], device=s.device)[None] < torch.tensor(kv_lens, device=s.device)[:, None]
        s = s.masked_fill(~keep[:, None, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None])
    return p @ v, lse, p


def _bounds(q, k, v, o, p, go, gl, e_o=HALF):
    """Error bounds of (dq, dk, dv), element by element."""
    n = q.shape[2] // k.shape[2]
    kd, vd = (t.transpose(1, 2).repeat_interleave(n, dim=1).abs() for t in (k, v))
    do, qd = go.abs(), q.transpose(1, 2).abs()
    oo = (do * o.abs()).sum(-1, keepdim=True)
    mag = do @ vd.transpose(2, 3) + oo + gl.abs()[..., None]
    ds = p * ((go @ v.transpose(1, 2).repeat_interleave(n, dim=1).transpose(2, 3) - (go * o).sum(-1, keepdim=True)) + gl[..., None])
    e = ds.abs() * (HALF + 2.0**-18) + p * (128 * 2.0**-24 * mag + e_o * oo)
    acc = 1 + max(q.shape[1] * n, k.shape[1]) * 2.0**-24 / HALF
    fold = lambda t: t.unflatten(1, (k.shape[2], n)).sum(2).transpose(1, 2)
    return ((SCALE * acc * e @ kd).transpose(1, 2), fold(SCALE * acc * e.transpose(2, 3) @ qd),
            fold((p * (acc * HALF + 2.0**-18)).transpose(2, 3) @ do))


def _check(got, want, bound):
    for name, x, y, e in zip(("dq", "dk", "dv"), got, want, bound):
        assert torch.isfinite(x).all(), name
        assert ((x.double() - y).abs() <= e + HALF * y.abs() + 1e-30).all(), name


@pytest.mark.parametrize("b,sq,skv,hq,hkv,kv_lens", [(1, 1, 1, 1, 1, None), (1, 257, 130, 2, 2, None), (2, 300, 513, 4, 2, None),
                                                     (2, 77, 200, 2, 1, [131, 1]), (1, 640, 64, 3, 1, None)])
@pytest.mark.parametrize("with_o", [True, False])
def test_against_definition(pkg, dev, b, sq, skv, hq, hkv, kv_lens, with_o):
    q, k, v, go, gl = _make(dev, b, sq, skv, hq, hkv, sq + skv)
    if not with_o:
        go = torch.zeros_like(go)
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    o, lse, p = _definition(*leaves, kv_lens)
    want = torch.autograd.grad((o * go.double()).sum() + (lse * gl.double()).sum(), leaves)
    with torch.no_grad():
        bound = _bounds(*(t.detach() for t in leaves), o, p, go.double(), gl.double())
        lse32 = _layout(lse)
        args = (go, q, k, v, o.to(torch.bfloat16), lse32)
        got = pkg.attention_bwd(*args, kv_lens=kv_lens, grad_lse=_layout(gl, math.nan))  # what lies behind the rows is not read
        _check(got, want, bound)
        plain = pkg.attention_bwd(*args, kv_lens=kv_lens)
        zero = pkg.attention_bwd(*args, kv_lens=kv_lens, grad_lse=torch.zeros_like(lse32))
        assert all(torch.equal(x, y) for x, y in zip(plain, zero))


def test_rows_without_probabilities(pkg, dev):
    """A row whose lse is -inf takes no gradient, whatever its grad_lse holds."""
    q, k, v, go, gl = _make(dev, 1, 200, 150, 2, 2, 5)
    with torch.no_grad():
        o, lse, _ = _definition(q.double(), k.double(), v.double())
        lse[:, :, 3] = -math.inf
        o[:, :, 3] = 0
        a = (go, q, k, v, o.to(torch.bfloat16), _layout(lse))
        gl[:, :, 3] = math.nan
        got = pkg.attention_bwd(*a, grad_lse=_layout(gl))
        gl[:, :, 3] = 0
        want = pkg.attention_bwd(*a, grad_lse=_layout(gl))
    assert all(torch.isfinite(x).all() and torch.equal(x, y) for x, y in zip(got, want))
    assert not got[0][:, 3].any()


def test_parts_merged_by_their_lse(pkg, dev):
    """Attention over two parts of the keys, merged by their lse, has the gradients of attention over all of them."""
    q, k, v, go, _ = _make(dev, 1, 200, 300, 2, 1, 9)
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad((_definition(*leaves)[0] * go.double()).sum(), leaves)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    fwd = torch.ops.b200omni.attention_fwd
    (o1, l1), (o2, l2) = fwd(q, k[:, :131], v[:, :131]), fwd(q, k[:, 131:], v[:, 131:])
    rows = lambda l: l.transpose(2, 3).flatten(2)[..., :200]
    w = torch.sigmoid(rows(l1) - rows(l2))[..., None]
    got = torch.autograd.grad((o1.float() * w + o2.float() * (1 - w)) * go.float(), (q, k, v), torch.ones_like(o1, dtype=torch.float32))
    # each part's P and o are off by 2 and 3 half steps more (bf16 probabilities summed under the norms' bound), its gradients are
    # rounded once by themselves and dq once more as their sum; grad_lse is formed from the parts' o, off by 3 half steps of theirs
    with torch.no_grad():
        qd, kd, vd = (t.detach() for t in leaves)
        n, total = 2, None
        for a, b in ((0, 131), (131, 300)):
            ws = w.double() if a == 0 else 1 - w.double()
            o, _, p = _definition(qd, kd[:, a:b], vd[:, a:b])
            # dS of the part = w P (dP - delta_part + grad_lse / w): magnitudes with |o1 - o2| through both parts' |o|
            other = _definition(qd, *((kd[:, 131:], vd[:, 131:]) if a == 0 else (kd[:, :131], vd[:, :131])))[0]
            mag_o = p @ vd[:, a:b].abs().transpose(1, 2).repeat_interleave(n, dim=1)
            d = go.double()
            gl = ((d * (o - other)).sum(-1, keepdim=True) * (1 - ws))[..., 0] * ws[..., 0]
            bq, bk, bv = _bounds(qd, kd[:, a:b], vd[:, a:b], mag_o, p, ws * d, gl, e_o=8 * HALF)
            e_gl = 8 * HALF * (d.abs() * (o.abs() + other.abs() + mag_o)).sum(-1, keepdim=True) * ws
            # the part's grad_o, w go, is rounded to bf16
            e_gl = e_gl + HALF * (ws * d).abs() @ vd[:, a:b].abs().transpose(1, 2).repeat_interleave(n, dim=1).transpose(2, 3)
            kk = kd[:, a:b].abs().transpose(1, 2).repeat_interleave(n, dim=1)
            bq = 4 * bq + (SCALE * (p * e_gl) @ kk).transpose(1, 2)
            bk = 4 * bk + (SCALE * (p * e_gl).transpose(2, 3) @ qd.abs().transpose(1, 2)).unflatten(1, (1, n)).sum(2).transpose(1, 2)
            bv = 4 * bv
            total = (bq, [bk], [bv]) if total is None else (total[0] + bq, total[1] + [bk], total[2] + [bv])
        bound = (total[0] + HALF * want[0].abs() * 2, torch.cat(total[1], 1), torch.cat(total[2], 1))
    _check(got, want, bound)


def test_lse_alone(pkg, dev):
    q, k, v, _, gl = _make(dev, 1, 130, 70, 2, 2, 11)
    for t in (q, k, v):
        t.requires_grad_(True)
    lse = torch.ops.b200omni.attention_fwd(q, k, v)[1]
    got = torch.autograd.grad((lse.transpose(2, 3).flatten(2)[..., :130] * gl).sum(), (q, k, v))
    assert not got[2].any() and got[0].any() and got[1].any()
