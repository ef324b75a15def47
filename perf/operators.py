"""What is measured of the trainable attention sub-layer: the attention's backward pass, rotary positions with
several axes, and the norms before and after a block fused with its gate and residual.

Each case is one pass through one operator. ``run`` computes it in plain torch (fp32, rounded once at the end) or,
where ``own`` is set, calls the framework. ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import importlib
import math

import torch

own = False

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
LOG = math.log

# ------------------------------------------------------------------ cases


def _attn(name, b, sq, skv, hq, hkv, q_lens="", kv_lens="", fused=False):
    """q_lens / kv_lens: comma-separated token counts per batch element ("" = whole rows); fused: q, k, v are column
    slices of one projection output."""
    return {"name": name, "op": "attention_bwd", "b": b, "sq": sq, "skv": skv, "hq": hq, "hkv": hkv, "q_lens": q_lens,
            "kv_lens": kv_lens, "fused": fused}


def _rope(name, b, s, hq, hk, axes, pairing="interleaved", dtype="bf16", inverse=False, positions="grid", theta=10000.0):
    return {"name": name, "op": "rotary", "b": b, "s": s, "hq": hq, "hk": hk, "axes": axes, "pairing": pairing,
            "dtype": dtype, "inverse": inverse, "positions": positions, "theta": theta}


def _norm(name, b, s, h, backward, post="rms_norm", norm="layer_norm", per_batch=True):
    return {"name": name, "op": "norm_bwd" if backward else "norm_fwd", "b": b, "s": s, "h": h, "post": post, "norm": norm,
            "per_batch": per_batch}


def listed():
    return [
        # the smallest call: a short clip's last, uneven chunk; latency counts
        _attn("attn_bwd_tiny", 1, 77, 77, 4, 4),
        # one layer's self-attention at 4096 tokens and all 40 heads, q / k / v inside the fused projection
        _attn("attn_bwd_s4096_h40", 1, 4096, 4096, 40, 40, fused=True),
        # a 480p clip's 32760 tokens, one group of 8 heads
        _attn("attn_bwd_s32760_h8", 1, 32760, 32760, 8, 8),
        # the same clip's cross-attention to 512 text tokens (a quarter of its tokens on this device)
        _attn("attn_bwd_cross_text", 1, 8190, 512, 40, 40),
        # a padded batch of uneven clips with shared key heads, one of them empty
        _attn("attn_bwd_padded_shared", 3, 1531, 1531, 12, 4, q_lens="1531,700,0", kv_lens="1531,700,0"),
        # rotary positions of a whole 480p clip: 21 frames of 30 x 52 patches
        _rope("rotary_clip_fwd", 1, 32760, 40, 40, "44,42,42"),
        # its gradient, two uneven images, rotate-half pairs, shared key heads
        _rope("rotary_bwd_images", 2, 1001, 24, 8, "16,56,56", pairing="half", inverse=True, positions="float"),
        # one token at a far position, in 32 bits
        _rope("rotary_token", 1, 1, 40, 40, "44,42,42", dtype="fp32", positions="far"),
        # the norms around a block at 32760 tokens of width 5120, forward and backward
        _norm("norm_fwd_clip", 1, 32760, 5120, False),
        _norm("norm_bwd_clip", 1, 32760, 5120, True),
        # a small batch of two at an odd length, width 1536
        _norm("norm_bwd_odd", 2, 333, 1536, True, post="layer_norm", norm="rms_norm"),
        # a handful of tokens
        _norm("norm_fwd_tokens", 1, 5, 5120, False, post="rms_norm", norm="rms_norm", per_batch=False),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(LOG(lo), LOG(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "norm_fwd", "norm_bwd"])
    if op == "attention":
        most = 8 * 32760 * 32760  # the largest listed case's query-key pairs
        b = rng.randint(1, 3)
        hkv, group = rng.choice([1, 2, 4, 5, 8, 10, 12, 40]), rng.choice([1, 1, 1, 2, 3])
        sq = _spread(rng, 1, 32760)
        skv = sq if rng.random() < 0.6 else _spread(rng, 1, 32760)
        while b * hkv * group * sq * skv > most or b * hkv * group * max(sq, skv) > 40 * 32760:
            sq, skv = max(1, sq * 3 // 4), max(1, skv * 3 // 4)
        q_lens = kv_lens = ""
        if rng.random() < 0.3:
            q_lens = ",".join(str(rng.randint(0, sq)) for _ in range(b))
            kv_lens = ",".join(str(rng.randint(0, skv)) for _ in range(b))
        c = _attn("", b, sq, skv, hkv * group, hkv, q_lens, kv_lens, fused=sq == skv and rng.random() < 0.5)
    elif op == "rotary":
        axes = rng.choice(["44,42,42", "16,56,56", "32,48,48", "8,28,28", "64,64", "24,20,20", "64"])
        b, hk, group = rng.randint(1, 3), rng.choice([1, 2, 5, 8, 12, 40]), rng.choice([1, 1, 3])
        s = _spread(rng, 1, 32760)
        while b * s * hk * (group + 1) > 80 * 32760:
            s = max(1, s * 3 // 4)
        c = _rope("", b, s, hk * group, hk, axes, rng.choice(["interleaved", "half"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                  rng.random() < 0.5, rng.choice(["grid", "float", "far"]), rng.choice([10000.0, 256.0, 1000000.0]))
    else:
        h = 8 * _spread(rng, 8, 1024)
        b, s = rng.randint(1, 3), _spread(rng, 1, 32760)
        while b * s * h > 32760 * 5120:
            s = max(1, s * 3 // 4)
        c = _norm("", b, s, h, op == "norm_bwd", rng.choice(["rms_norm", "layer_norm", "none"]),
                  rng.choice(["layer_norm", "rms_norm"]), rng.random() < 0.7)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs


def _lens(text, n, b):
    return [int(v) for v in text.split(",")] if text else [n] * b


def _axes(case):
    return tuple(int(v) for v in case["axes"].split(","))


def _valid(lens, n, device):
    return torch.arange(n, device=device)[None, :] < torch.tensor(lens, device=device)[:, None]


def _prepare_attention(c, gen):
    b, sq, skv, hq, hkv, d = c["b"], c["sq"], c["skv"], c["hq"], c["hkv"], 128
    if c["fused"]:
        qkv = torch.randn(b, sq, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(BF16)
        q, k, v = (t.unflatten(2, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=2))
    else:
        q, k, v = (torch.randn(b, s, h, d, generator=gen, device="cuda").to(BF16) for s, h in ((sq, hq), (skv, hkv), (skv, hkv)))
    # a gradient of the size that a mean over tokens leaves
    grad_o = (torch.randn(b, hq, sq, d, generator=gen, device="cuda") / 64).to(BF16)
    q_lens, kv_lens = _lens(c["q_lens"], sq, b), _lens(c["kv_lens"], skv, b)
    scale = 1.0 / math.sqrt(d)
    # the forward pass's output and log-sum-exp, in the layouts that the framework's forward returns
    o = torch.zeros(b, hq, sq, d, dtype=BF16, device="cuda")
    rows = torch.full((b, hq, sq), -math.inf, device="cuda")
    for i in range(b):
        if q_lens[i] and kv_lens[i]:
            for h in range(hq):
                s = (q[i, : q_lens[i], h].float() @ k[i, : kv_lens[i], h * hkv // hq].float().T) * scale
                l = torch.logsumexp(s, dim=-1)
                o[i, h, : q_lens[i]] = (s.sub_(l[:, None]).exp_() @ v[i, : kv_lens[i], h * hkv // hq].float()).to(BF16)
                rows[i, h, : q_lens[i]] = l
    groups = -(-sq // 128)
    lse = torch.zeros(b, hq, groups * 128, device="cuda")
    lse[:, :, :sq] = rows
    lse = lse.reshape(b, hq, groups, 128).transpose(2, 3).contiguous()
    return {"case": c, "q": q, "k": k, "v": v, "o": o, "lse": lse, "grad_o": grad_o, "scale": scale, "q_lens": q_lens,
            "kv_lens": kv_lens}


def _grid_positions(n):
    """(frame, row, column) of the first n patches of frames of 30 x 52."""
    i = torch.arange(n, dtype=torch.int32, device="cuda")
    return torch.stack([i // 1560, i // 52 % 30, i % 52], dim=-1)


def _prepare_rotary(c, gen):
    axes = _axes(c)
    d, b, s = sum(axes), c["b"], c["s"]
    qkv = torch.randn(b, s, (c["hq"] + 2 * c["hk"]) * d, generator=gen, device="cuda").to(DTYPES[c["dtype"]])
    q, k, _ = (t.unflatten(2, (-1, d)) for t in qkv.split([c["hq"] * d, c["hk"] * d, c["hk"] * d], dim=2))
    if c["positions"] == "grid":  # whole patches, shared by the batch
        pos = _grid_positions(s)[:, -len(axes):].contiguous()
    elif c["positions"] == "far":  # frames and tokens of a long stream
        pos = torch.randint(0, 1 << 20, (b, s, len(axes)), generator=gen, device="cuda", dtype=torch.int32)
    else:  # interpolated positions
        pos = torch.rand(b, s, len(axes), generator=gen, device="cuda") * 96.0
    return {"case": c, "q": q, "k": k, "positions": pos, "axes": axes}


def _prepare_norm(c, gen):
    b, s, h = c["b"], c["s"], c["h"]
    mk = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    vec = (b, 1, h) if c["per_batch"] else (h,)
    # sub-layer outputs and residual streams have means and scales of their own
    st = {"case": c, "x": (0.3 + 0.8 * mk(b, s, h)).to(BF16), "residual": (2.0 * mk(b, s, h) - 0.2).to(BF16), "gate": 0.5 * mk(*vec),
          "mul": 1 + 0.2 * mk(*vec), "add": 0.2 * mk(*vec), "weight": None if c["post"] == "none" else 1 + 0.2 * mk(h), "eps": 1e-6}
    if c["op"] == "norm_bwd":
        st["grad_r"], st["grad_out"] = (mk(b, s, h) / 64).to(BF16), (mk(b, s, h) / 64).to(BF16)
        # the residual stream as the forward pass stored it
        y = _hat(st["x"].float(), c["post"], st["eps"])[0]
        st["residual_out"] = (st.pop("residual").float() + st["gate"] * (y if st["weight"] is None else y * st["weight"])).to(BF16)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "attention_bwd":
        return _prepare_attention(case, gen)
    if case["op"] == "rotary":
        return _prepare_rotary(case, gen)
    return _prepare_norm(case, gen)


# ------------------------------------------------------------------ plain forms


def _plain_attention(st):
    """dv = P^T dO, dS = P (dO V^T - rowsum(dO O)), dq = scale dS K, dk = scale dS^T Q with P = exp(scale Q K^T - lse)."""
    q, k, v, do, o = st["q"], st["k"], st["v"], st["grad_o"], st["o"]
    b, sq, hq, d = q.shape
    skv, hkv = k.shape[1:3]
    g = hq // hkv
    lse = st["lse"].transpose(2, 3).reshape(b, hq, -1)[:, :, :sq]
    keep = (_valid(st["q_lens"], sq, q.device)[:, :, None] & _valid(st["kv_lens"], skv, q.device)[:, None, :])[:, None]
    dq, dk, dv = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty(b, skv, hkv, d, dtype=BF16, device=q.device), torch.empty(
        b, skv, hkv, d, dtype=BF16, device=q.device)
    step = max(1, min(hkv, (1 << 30) // max(1, b * g * sq * skv)))  # key heads whose scores are held at once
    for h in range(0, hkv, step):
        n = min(step, hkv - h)
        qh, doh, oh = (t.float() for t in (q.transpose(1, 2)[:, h * g:(h + n) * g], do[:, h * g:(h + n) * g], o[:, h * g:(h + n) * g]))
        kh, vh = (t.transpose(1, 2)[:, h:h + n].float().repeat_interleave(g, dim=1) for t in (k, v))
        p = torch.where(keep, torch.exp(qh @ kh.transpose(2, 3) * st["scale"] - lse[:, h * g:(h + n) * g, :, None]), 0.0)
        dvh = p.transpose(2, 3) @ doh
        ds = p * (doh @ vh.transpose(2, 3) - (doh * oh).sum(-1, keepdim=True))
        dq[:, :, h * g:(h + n) * g] = (ds @ kh * st["scale"]).transpose(1, 2)
        dk[:, :, h:h + n] = (ds.transpose(2, 3) @ qh * st["scale"]).unflatten(1, (n, g)).sum(2).transpose(1, 2)
        dv[:, :, h:h + n] = dvh.unflatten(1, (n, g)).sum(2).transpose(1, 2)
    return dq, dk, dv


def _plain_rotary(st):
    c, axes = st["case"], st["axes"]
    freqs = torch.cat([c["theta"] ** (-torch.arange(0, n, 2, dtype=F64, device="cuda") / n) for n in axes])
    axis = torch.repeat_interleave(torch.arange(len(axes), device="cuda"), torch.tensor([n // 2 for n in axes], device="cuda"))
    angle = st["positions"].to(F64)[..., axis] * freqs  # [(b,) s, d / 2]
    if c["inverse"]:
        angle = -angle
    cos, sin = (t.float().unsqueeze(-2) for t in (angle.cos(), angle.sin()))
    half = c["pairing"] == "half"

    def turn(x):
        x1, x2 = x.float().chunk(2, dim=-1) if half else x.float().unflatten(-1, (-1, 2)).unbind(-1)
        y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
        return (torch.cat([y1, y2], dim=-1) if half else torch.stack([y1, y2], dim=-1).flatten(-2)).to(x.dtype)

    return turn(st["q"]), turn(st["k"])


def _hat(x, kind, eps):
    """(normalised x, 1 / its deviation) over the last axis."""
    if kind == "none":
        return x, 1.0
    if kind == "layer_norm":
        x = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * rstd, rstd


def _hat_grad(g, hat, rstd, kind):
    """The gradient behind _hat, given the gradient g of its result."""
    if kind == "none":
        return g
    out = g - hat * (g * hat).mean(-1, keepdim=True)
    if kind == "layer_norm":
        out = out - g.mean(-1, keepdim=True)
    return out * rstd


def _plain_norm_fwd(st):
    c = st["case"]
    y = _hat(st["x"].float(), c["post"], st["eps"])[0]
    if st["weight"] is not None:
        y = y * st["weight"]
    r = st["residual"].float() + st["gate"] * y
    return r.to(BF16), (_hat(r, c["norm"], st["eps"])[0] * st["mul"] + st["add"]).to(BF16)


def _plain_norm_bwd(st):
    c, over = st["case"], (1,) if st["case"]["per_batch"] else (0, 1)
    total = lambda t: t.sum(over, keepdim=c["per_batch"])  # noqa: E731
    n, rstd = _hat(st["residual_out"].float(), c["norm"], st["eps"])
    go = st["grad_out"].float()
    dr = st["grad_r"].float() + _hat_grad(go * st["mul"], n, rstd, c["norm"])
    y, rstd_x = _hat(st["x"].float(), c["post"], st["eps"])
    w = 1.0 if st["weight"] is None else st["weight"]
    dx = _hat_grad(dr * st["gate"] * w, y, rstd_x, c["post"])
    dw = () if st["weight"] is None else ((dr * st["gate"] * y).sum((0, 1)),)
    return (dx.to(BF16), dr.to(BF16), total(dr * y * w), total(go * n), total(go)) + dw


# ------------------------------------------------------------------ one pass


def _own(st):
    f = importlib.import_module("vllm-omni-neuron_b200")
    c = st["case"]
    if c["op"] == "attention_bwd":
        lens = {"q_lens": st["q_lens"], "kv_lens": st["kv_lens"]} if c["q_lens"] else {}
        return f.attention_bwd(st["grad_o"], st["q"], st["k"], st["v"], st["o"], st["lse"], st["scale"], **lens)
    if c["op"] == "rotary":
        return f.rotary_axes(st["q"], st["k"], st["positions"], st["axes"], theta=c["theta"], pairing=c["pairing"], inverse=c["inverse"])
    kinds = {"eps": st["eps"], "post_norm": c["post"], "post_weight": st["weight"], "norm_type": c["norm"]}
    if c["op"] == "norm_fwd":
        return f.sandwich_norm(st["x"], st["residual"], st["gate"], st["mul"], st["add"], **kinds)
    g = f.sandwich_norm_bwd(st["grad_r"], st["grad_out"], st["x"], st["residual_out"], st["gate"], st["mul"], st["add"], **kinds)
    return (g.x, g.residual, g.gate, g.mul, g.add) + (() if g.post_weight is None else (g.post_weight,))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "attention_bwd":
        return _plain_attention(state)
    if op == "rotary":
        return _plain_rotary(state)
    return _plain_norm_fwd(state) if op == "norm_fwd" else _plain_norm_bwd(state)


# ------------------------------------------------------------------ the cost that no implementation can avoid


def work(case):
    c = case
    if c["op"] == "attention_bwd":
        ql, kl = _lens(c["q_lens"], c["sq"], c["b"]), _lens(c["kv_lens"], c["skv"], c["b"])
        pairs = sum(x * y for x, y in zip(ql, kl))
        read = sum(ql) * c["hq"] * (3 * 256 + 4) + sum(kl) * c["hkv"] * 2 * 256  # q, o, grad_o, lse; k, v
        written = c["b"] * (c["sq"] * c["hq"] + 2 * c["skv"] * c["hkv"]) * 256  # dq, dk, dv
        return {"bytes": read + written, "flops": 5 * 2 * 128 * pairs * c["hq"]}
    if c["op"] == "rotary":
        axes = _axes(c)
        n = c["b"] * c["s"] * (c["hq"] + c["hk"]) * sum(axes)
        pos = c["s"] * (1 if c["positions"] == "grid" else c["b"]) * len(axes) * 4
        return {"bytes": 2 * n * (4 if c["dtype"] == "fp32" else 2) + pos, "flops": 3 * n}
    n, vecs = c["b"] * c["s"] * c["h"], (c["b"] if c["per_batch"] else 1) * c["h"] * 4
    w = 0 if c["post"] == "none" else 4 * c["h"]
    if c["op"] == "norm_fwd":
        return {"bytes": 8 * n + 3 * vecs + w, "flops": 12 * n}  # x, residual; residual_out, out
    return {"bytes": 12 * n + 5 * vecs + 2 * w, "flops": 30 * n}  # x, residual_out, two gradients; two gradients, sums


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_attention(st):
    b, sq, hq, d = st["q"].shape
    skv, hkv = st["k"].shape[1:3]
    out = [torch.zeros(b, n, h, d, dtype=F64, device="cuda") for n, h in ((sq, hq), (skv, hkv), (skv, hkv))]
    for i in range(b):
        m, n = st["q_lens"][i], st["kv_lens"][i]
        if not m or not n:
            continue
        for h in range(hq):
            a = h * hkv // hq
            q, k, v = st["q"][i, :m, h].double(), st["k"][i, :n, a].double(), st["v"][i, :n, a].double()
            o, do = st["o"][i, h, :m].double(), st["grad_o"][i, h, :m].double()
            logz = st["lse"][i, h].T.flatten()[:m].double()
            w = torch.einsum("md,nd->mn", q, k).mul_(st["scale"]).sub_(logz.unsqueeze(1)).exp_()
            out[2][i, :n, a] += torch.einsum("mn,md->nd", w, do)
            w.mul_(torch.einsum("md,nd->mn", do, v).sub_(torch.einsum("md,md->m", do, o).unsqueeze(1)))
            out[0][i, :m, h] = torch.einsum("mn,nd->md", w, k) * st["scale"]
            out[1][i, :n, a] += torch.einsum("mn,md->nd", w, q) * st["scale"]
    return tuple(out)


def _exact_rotary(st):
    c, axes = st["case"], st["axes"]
    d, sign = sum(axes), -1.0 if c["inverse"] else 1.0
    pos = st["positions"].double()
    outs = []
    for x in (st["q"], st["k"]):
        y, pair = torch.empty_like(x, dtype=F64, memory_format=torch.contiguous_format), 0
        for a, n in enumerate(axes):
            for i in range(n // 2):
                i1, i2 = (pair, pair + d // 2) if c["pairing"] == "half" else (2 * pair, 2 * pair + 1)
                turn = torch.polar(torch.ones_like(pos[..., a]), sign * pos[..., a] * c["theta"] ** (-2 * i / n)).unsqueeze(-1)
                z = torch.complex(x[..., i1].double(), x[..., i2].double()) * turn
                y[..., i1], y[..., i2] = z.real, z.imag
                pair += 1
        outs.append(y)
    return tuple(outs)


def _exact_norm(st, backward):
    """The forward from its definition; the gradients by 64-bit differentiation of it."""
    c = st["case"]
    need = lambda t: None if t is None else t.double().requires_grad_(backward)  # noqa: E731
    x, gate, mul, add, weight = (need(st[k]) for k in ("x", "gate", "mul", "add", "weight"))

    def normal(t, kind):
        if kind == "none":
            return t
        centre = t.mean(-1, keepdim=True) if kind == "layer_norm" else 0.0
        return (t - centre) / ((t - centre).square().mean(-1, keepdim=True) + st["eps"]).sqrt()

    branch = normal(x, c["post"])
    branch = gate * (branch if weight is None else branch * weight)
    if not backward:
        r = st["residual"].double() + branch
        return r, normal(r, c["norm"]) * mul + add
    r = st["residual_out"].double().requires_grad_(True)  # the stream as the forward pass stored it
    out = normal(r, c["norm"]) * mul + add
    leaves = [r, mul, add]
    dr, dmul, dadd = torch.autograd.grad(out, leaves, st["grad_out"].double())
    dr = dr + st["grad_r"].double()
    leaves = [x, gate] + ([] if weight is None else [weight])
    dx, dgate, *dw = torch.autograd.grad(branch, leaves, dr)
    return (dx, dr, dgate, dmul, dadd, *dw)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention_bwd":
        return _exact_attention(st)
    if case["op"] == "rotary":
        return _exact_rotary(st)
    return _exact_norm(st, case["op"] == "norm_bwd")
