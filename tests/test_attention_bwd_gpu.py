"""The attention's gradients against the definition in 64 bits (B200 only).

Tolerances count roundings: P and dS enter the tensor cores as bf16 (2^-8 relative each), the results are rounded to
bf16 once (2^-8), the products are sums of 128 terms in fp32 (128 * 2^-24 of the sum of their magnitudes), and the
exponential's argument and value carry a few 2^-24 (2^-18 relative in all for arguments below 32). Every bound is formed
from the magnitudes in 64 bits, element by element."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0**-8  # half a step of bf16, relative
ACC = 128 * 2.0**-24
EXP = 2.0**-18


def _lse_layout(rows):
    b, h, s = rows.shape
    g = -(-s // 128)
    full = torch.zeros(b, h, g * 128, dtype=torch.float32, device=rows.device)
    full[:, :, :s] = rows.float()
    return full.reshape(b, h, g, 128).transpose(2, 3).contiguous()


def _inputs(dev, b, sq, skv, hq, hkv, seed, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)
    q, k, v = mk(b, sq, hq, 128) * scale_q, mk(b, skv, hkv, 128), mk(b, skv, hkv, 128) + 0.25
    go = mk(b, hq, sq, 128) * 0.05
    return [t.to(torch.bfloat16).to(dev) for t in (q, k, v, go)]


def _scores(q, k, scale, q_lens, kv_lens):
    b, sq, hq, _ = q.shape
    skv, hkv = k.shape[1:3]
    kk = k.double().transpose(1, 2).repeat_interleave(hq // hkv, dim=1)
    s = scale * q.double().transpose(1, 2) @ kk.transpose(2, 3)
    ql = torch.tensor(q_lens or [sq] * b, device=q.device)
    kl = torch.tensor(kv_lens or [skv] * b, device=q.device)
    keep = (torch.arange(sq, device=q.device)[None] < ql[:, None])[:, None, :, None] & (
        torch.arange(skv, device=q.device)[None] < kl[:, None])[:, None, None, :]
    return s, keep


def _forward(q, k, v, scale, q_lens=None, kv_lens=None):
    """(o fp64 [b, h, s, d], lse rows fp64): 0 and -inf where nothing is kept."""
    hq, hkv = q.shape[2], k.shape[2]
    s, keep = _scores(q, k, scale, q_lens, kv_lens)
    s = s.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    p = torch.where(keep, torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None]), 0.0)
    return p @ v.double().transpose(1, 2).repeat_interleave(hq // hkv, dim=1), lse


def _grads(q, k, v, o, lse, go, scale, q_lens=None, kv_lens=None, e_p=0.0, e_o=0.0):
    """((dq, dk, dv), their error bounds) in fp64; e_p / e_o: further relative errors of P and o."""
    hq, hkv = q.shape[2], k.shape[2]
    g = hq // hkv
    s, keep = _scores(q, k, scale, q_lens, kv_lens)
    keep = keep & ~lse.isinf()[..., None]
    p = torch.where(keep, torch.exp(s - torch.where(lse.isinf(), 0.0, lse.double())[..., None]), 0.0)
    qd, do, od = q.double().transpose(1, 2), go.double(), o.double()
    kd, vd = (t.double().transpose(1, 2).repeat_interleave(g, dim=1) for t in (k, v))
    delta = (do * od).sum(-1, keepdim=True)
    ds = p * (do @ vd.transpose(2, 3) - delta)
    mag = do.abs() @ vd.abs().transpose(2, 3) + (do.abs() * od.abs()).sum(-1, keepdim=True)
    e_ds = ds.abs() * (HALF + EXP + e_p) + p * (ACC * mag + e_o * (do.abs() * od.abs()).sum(-1, keepdim=True))
    fold = lambda t: t.unflatten(1, (hkv, g)).sum(2).transpose(1, 2)
    dq = (scale * ds @ kd).transpose(1, 2)
    dk, dv = fold(scale * ds.transpose(2, 3) @ qd), fold(p.transpose(2, 3) @ do)
    n = max(q.shape[1] * g, k.shape[1])
    acc = 1 + n * 2.0**-24 / HALF  # fp32 sums of the products
    b_dq = (scale * (acc * e_ds) @ kd.abs()).transpose(1, 2) + HALF * dq.abs()
    b_dk = fold(scale * (acc * e_ds).transpose(2, 3) @ qd.abs()) + HALF * dk.abs()
    b_dv = fold((p * (acc * HALF + EXP + e_p)).transpose(2, 3) @ do.abs()) + HALF * dv.abs()
    return (dq, dk, dv), tuple(b + 1e-30 for b in (b_dq, b_dk, b_dv))


def _check(got, ref, bound, what=""):
    for name, x, y, e in zip(("dq", "dk", "dv"), got, ref, bound):
        assert x.shape == y.shape and x.dtype == torch.bfloat16 and x.is_contiguous(), name
        assert torch.isfinite(x).all(), f"{what} {name} has non-finite values"
        over = ((x.double() - y).abs() / e).max().item()
        assert over <= 1.0, f"{what} {name}: {over:.3f} of the bound"


def _status():
    from importlib import import_module

    return import_module("vllm-omni-neuron_b200._lib").device_status()


def _run(pkg, q, k, v, go, scale=None, q_lens=None, kv_lens=None):
    sc = 1 / math.sqrt(128) if scale is None else scale
    o, lse = _forward(q, k, v, sc, q_lens, kv_lens)
    o = o.to(torch.bfloat16)
    got = pkg.attention_bwd(go, q, k, v, o, _lse_layout(lse), scale, q_lens=q_lens, kv_lens=kv_lens)
    torch.cuda.synchronize()
    assert _status() == 0
    return got, _grads(q, k, v, o, lse.float(), go, sc, q_lens, kv_lens)


@pytest.mark.parametrize(
    "b,sq,skv,hq,hkv",
    [
        (1, 128, 128, 1, 1),
        (1, 1, 1, 1, 1),
        (1, 256, 256, 2, 2),
        (1, 129, 1, 2, 1),
        (1, 1, 1000, 3, 3),
        (1, 1000, 1, 2, 2),
        (2, 77, 200, 4, 2),
        (1, 513, 640, 2, 2),
        (2, 300, 300, 6, 2),
        (1, 2048, 77, 1, 1),
        (1, 64, 3001, 1, 1),
        (1, 700, 512, 3, 1),
    ],
)
def test_against_definition(pkg, dev, b, sq, skv, hq, hkv):
    got, want = _run(pkg, *_inputs(dev, b, sq, skv, hq, hkv, sq + skv))
    _check(got, *want)


@pytest.mark.parametrize("scale", [0.02, 0.25, -0.05])
def test_scales(pkg, dev, scale):
    got, want = _run(pkg, *_inputs(dev, 1, 200, 333, 2, 2, 5), scale=scale)
    _check(got, *want)


def test_lengths_ignore_what_lies_behind(pkg, dev):
    q, k, v, go = _inputs(dev, 4, 300, 400, 4, 2, 11)
    q_lens, kv_lens = [300, 77, 0, 129], [400, 0, 131, 257]
    got, want = _run(pkg, q, k, v, go, q_lens=q_lens, kv_lens=kv_lens)
    _check(got, *want)
    for i in range(4):
        assert not got[0][i, q_lens[i]:].any() and not got[1][i, kv_lens[i]:].any() and not got[2][i, kv_lens[i]:].any()
    o, lse = _forward(q, k, v, 1 / math.sqrt(128), q_lens, kv_lens)
    o = o.to(torch.bfloat16)
    for i in range(4):  # the same bits with NaN and infinities behind the ends
        q[i, q_lens[i]:] = math.nan
        go[i, :, q_lens[i]:] = math.inf
        o[i, :, q_lens[i]:] = math.nan
        k[i, kv_lens[i]:] = math.nan
        v[i, kv_lens[i]:] = -math.inf
        lse[i, :, q_lens[i]:] = math.nan
    again = pkg.attention_bwd(go, q, k, v, o, _lse_layout(lse), q_lens=q_lens, kv_lens=kv_lens)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_more_sequences_than_one_launch_holds(pkg, dev):
    b = 19
    q, k, v, go = _inputs(dev, b, 40, 50, 2, 1, 12)
    q_lens, kv_lens = [(7 * i) % 41 for i in range(b)], [(11 * i + 3) % 51 for i in range(b)]
    got, want = _run(pkg, q, k, v, go, q_lens=q_lens, kv_lens=kv_lens)
    _check(got, *want)
    got, want = _run(pkg, q, k, v, go, kv_lens=kv_lens)
    _check(got, *want)


@pytest.mark.parametrize("sq,skv,hq,hkv,q_lens,kv_lens", [
    (7700, 200, 22, 11, None, None),  # 31 tiles of 256 queries a head: several a CTA pair, the last group short
    (8190, 512, 40, 40, None, None),
    (5000, 250, 20, 20, [5000, 1300, 0], [250, 100, 250]),  # walks of two steps, of one, of none
])
def test_short_walks(pkg, dev, sq, skv, hq, hkv, q_lens, kv_lens):
    """Many queries, few keys: a pair takes several query tiles one after the other."""
    b = len(q_lens) if q_lens else 1
    q, k, v, go = _inputs(dev, b, sq, skv, hq, hkv, 22)
    sc = 1 / math.sqrt(128)
    o = torch.zeros(b, hq, sq, 128, dtype=torch.bfloat16, device=dev)
    lse = torch.full((b, hq, sq), -math.inf, device=dev, dtype=torch.float64)
    g = hq // hkv
    for h in range(hkv):  # the reference head by head
        oo, ll = _forward(q[:, :, h * g:(h + 1) * g], k[:, :, h:h + 1], v[:, :, h:h + 1], sc, q_lens, kv_lens)
        o[:, h * g:(h + 1) * g], lse[:, h * g:(h + 1) * g] = oo.to(torch.bfloat16), ll
    got = pkg.attention_bwd(go, q, k, v, o, _lse_layout(lse), q_lens=q_lens, kv_lens=kv_lens)
    torch.cuda.synchronize()
    assert _status() == 0
    for h in range(hkv):
        part = [t[:, :, h * g:(h + 1) * g] if i == 0 else t[:, :, h:h + 1] for i, t in enumerate(got)]
        want, bound = _grads(q[:, :, h * g:(h + 1) * g], k[:, :, h:h + 1], v[:, :, h:h + 1], o[:, h * g:(h + 1) * g],
                             lse[:, h * g:(h + 1) * g].float(), go[:, h * g:(h + 1) * g], sc, q_lens, kv_lens)
        _check([t.contiguous() for t in part], want, bound, f"head {h}")


def test_rows_without_probabilities(pkg, dev):
    q, k, v, go = _inputs(dev, 1, 150, 150, 1, 1, 13)
    sc = 1 / math.sqrt(128)
    o, lse = _forward(q, k, v, sc)
    o = o.to(torch.bfloat16)
    lse[:, :, 40:60] = -math.inf
    got = pkg.attention_bwd(go, q, k, v, o, _lse_layout(lse), sc)
    _check(got, *_grads(q, k, v, o, lse.float(), go, sc))
    assert not got[0][:, 40:60].any()


def test_views(pkg, dev):
    """Column slices of a fused projection, head-major memory, broadcast heads and an odd storage offset."""
    b, s, h = 2, 193, 3
    q, k, v, go = _inputs(dev, b, s, s, h, h, 14)
    base, want = _run(pkg, q, k, v, go)
    _check(base, *want)
    sc = 1 / math.sqrt(128)
    o, lse = _forward(q, k, v, sc)
    o, lse = o.to(torch.bfloat16), _lse_layout(lse)
    fused = torch.cat([t.flatten(2) for t in (q, k, v)], dim=-1)
    qf, kf, vf = (t.unflatten(2, (h, 128)) for t in fused.chunk(3, dim=-1))
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    gt = go.transpose(1, 2).contiguous().transpose(1, 2)
    ot = o.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(k.numel() + 3, dtype=k.dtype, device=dev)[3:].view(k.shape).copy_(k)
    for args in ((go, qf, kf, vf, o), (gt, qh, k, v, ot), (go, q, odd, v, o)):
        assert all(torch.equal(x, y) for x, y in zip(base, pkg.attention_bwd(*args, lse)))
    one = v[:, :, :1].expand(b, s, h, 128)  # stride 0: as a copy of it
    o1, l1 = _forward(q, k, one, sc)
    args = (o1.to(torch.bfloat16), _lse_layout(l1))
    a, c = pkg.attention_bwd(go, q, k, one, *args), pkg.attention_bwd(go, q, k, one.contiguous(), *args)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_far_offsets(pkg, dev):
    """Element offsets past 2^31: a token stride of 2^23 over 300 tokens."""
    q, k, v, go = _inputs(dev, 1, 300, 300, 1, 1, 15)
    base, want = _run(pkg, q, k, v, go)
    far = torch.empty_strided((1, 300, 1, 128), (300 << 23, 1 << 23, 128, 1), dtype=torch.bfloat16, device=dev)
    o, lse = _forward(q, k, v, 1 / math.sqrt(128))
    far.copy_(q)
    a = pkg.attention_bwd(go, far, k, v, o.to(torch.bfloat16), _lse_layout(lse))
    far.copy_(k)
    b = pkg.attention_bwd(go, q, far, v, o.to(torch.bfloat16), _lse_layout(lse))
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(base, a, b))


def test_parts_of_the_keys_add_up(pkg, dev):
    """The ring's use: each part of the keys with the whole sequence's o and lse."""
    q, k, v, go = _inputs(dev, 1, 260, 500, 2, 2, 16)
    sc = 1 / math.sqrt(128)
    o, lse = _forward(q, k, v, sc)
    o = o.to(torch.bfloat16)
    (dq, dk, dv), (b_dq, b_dk, b_dv) = _grads(q, k, v, o, lse.float(), go, sc)
    parts = [pkg.attention_bwd(go, q, k[:, a:b], v[:, a:b], o, _lse_layout(lse), sc) for a, b in ((0, 131), (131, 500))]
    total = parts[0][0].double() + parts[1][0].double()
    assert ((total - dq).abs() <= b_dq + HALF * (parts[0][0].double().abs() + parts[1][0].double().abs())).all()
    assert ((torch.cat([p[1] for p in parts], 1).double() - dk).abs() <= b_dk).all()
    assert ((torch.cat([p[2] for p in parts], 1).double() - dv).abs() <= b_dv).all()


def test_same_bits_every_time_and_on_another_stream(pkg, dev):
    q, k, v, go = _inputs(dev, 1, 900, 1100, 3, 1, 17)
    first, _ = _run(pkg, q, k, v, go)
    o, lse = _forward(q, k, v, 1 / math.sqrt(128))
    o, lse = o.to(torch.bfloat16), _lse_layout(lse)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        runs = [pkg.attention_bwd(go, q, k, v, o, lse) for _ in range(3)]
    here = [pkg.attention_bwd(go, q, k, v, o, lse) for _ in range(3)]  # beside the other stream's
    torch.cuda.synchronize()
    for r in runs + here:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed(pkg, dev):
    q, k, v, go = _inputs(dev, 1, 300, 300, 2, 2, 18)
    sc = 1 / math.sqrt(128)
    o, lse = _forward(q, k, v, sc)
    o, lse = o.to(torch.bfloat16), _lse_layout(lse)
    pkg.attention_bwd(go, q, k, v, o, lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.attention_bwd(go, q, k, v, o, lse)
    q2, k2, v2, go2 = _inputs(dev, 1, 300, 300, 2, 2, 19)
    o2, l2 = _forward(q2, k2, v2, sc)
    for dst, src in ((q, q2), (k, k2), (v, v2), (go, go2), (o, o2.to(torch.bfloat16)), (lse, _lse_layout(l2))):
        dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    _check(out, *_grads(q, k, v, o, l2.float(), go, sc))


@pytest.mark.parametrize("b,sq,skv,hq,hkv,lens", [(1, 333, 333, 2, 2, None), (2, 200, 512, 4, 2, None),
                                                  (3, 140, 140, 2, 1, [140, 3, 0])])
def test_differentiable_form(pkg, dev, b, sq, skv, hq, hkv, lens):
    """wan_attention forward and backward. Its o is off by HALF and its lse, summed from bf16 probabilities under the
    Cauchy-Schwarz bound, by at most HALF, so P carries HALF more and o, whose P is normalised by that sum, 3 HALF."""
    q, k, v, go = _inputs(dev, b, sq, skv, hq, hkv, 20)
    sc = 1 / math.sqrt(128)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = pkg.wan_attention(q, k, v, q_lens=lens, kv_lens=lens)
    assert o.shape == (b, hq, sq, 128)
    grads = torch.autograd.grad(o, (q, k, v), go)
    with torch.no_grad():
        ro, rl = _forward(q, k, v, sc, lens, lens)
        s, keep = _scores(q, k, sc, lens, lens)
        p = torch.where(keep & ~rl.isinf()[..., None], torch.exp(s - torch.where(rl.isinf(), 0.0, rl)[..., None]), 0.0)
        mag = p @ v.double().abs().transpose(1, 2).repeat_interleave(hq // hkv, dim=1)
        assert ((o.double() - ro).abs() <= 3 * HALF * mag + HALF * ro.abs() + 1e-30).all()
        # o's error, relative to its magnitudes, moves delta: bound it through mag
        e_delta = (go.double().abs() * (3 * HALF * mag + HALF * ro.abs())).sum(-1, keepdim=True)
        want, bound = _grads(q, k, v, ro, rl, go, sc, lens, lens, e_p=HALF)
        kd = k.double().transpose(1, 2).repeat_interleave(hq // hkv, dim=1).abs()
        more = p * e_delta
        fold = lambda t: t.unflatten(1, (hkv, hq // hkv)).sum(2).transpose(1, 2)
        bound = (bound[0] + (sc * more @ kd).transpose(1, 2),
                 bound[1] + fold(sc * more.transpose(2, 3) @ q.double().transpose(1, 2).abs()), bound[2])
        _check(grads, want, bound)
        if lens:
            for i, n in enumerate(lens):
                assert not o[i, :, n:].any()


def test_against_differences(pkg, dev):
    """The directional derivative along random directions, by central differences of the 64-bit forward."""
    q, k, v, go = _inputs(dev, 1, 70, 90, 2, 1, 21)
    got, want = _run(pkg, q, k, v, go)
    g = torch.Generator().manual_seed(3)
    sc, h = 1 / math.sqrt(128), 1e-5
    for i, t in enumerate((q, k, v)):
        u = torch.randn(t.shape, generator=g, dtype=torch.float64).to(dev)
        ends = []
        for e in (h, -h):
            args = [x.double() for x in (q, k, v)]
            args[i] = args[i] + e * u
            ends.append((_forward(*args, sc)[0] * go.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        # o is rounded to bf16 for delta: half a step of it moves delta, which the bound of _grads takes as given
        o = _forward(q, k, v, sc)[0]
        _, loose = _grads(q, k, v, o, _forward(q, k, v, sc)[1], go, sc, e_o=HALF)
        room = (loose[i] * u.abs()).sum() + 1e-6
        assert (got[i].double().mul(u).sum() - slope).abs() <= room
