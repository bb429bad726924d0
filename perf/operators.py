"""The operators of a decoder's training and serving around its attention and its loss, measured:
rotary positions (rope), per-head norms of queries and keys with the rotation in the same pass
(qk_norm_rope), and the softmax cross entropy of a linear head without its logits (linear_xent).

Each case is one pass through an operator's public entry points (gn_bwd's functions) or, with
`own` false, its plain form in torch.  Inputs are seeded and synthetic: activations N(0, 1),
upstream gradients N(0, 0.01), weights as the repository's benchmark draws them.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "grilly-next_amd"))

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # One new token for each of 32 running sequences, every one at its own far position of a
        # context stretched 32-fold (YaRN): a few hundred kilobytes, latency is all of it.
        dict(name="rope_token", kind="rope", dir="fwd", batch=32, seq=1, heads=24, dim=64, rot=64, mode="half",
             scaling="yarn", factor=32.0, start=100000, dtype="bf16"),
        # A long prompt's queries and keys (16 + 4 heads), half of each head rotated, an odd length.
        dict(name="rope_prompt", kind="rope", dir="fwd", batch=1, seq=30001, heads=20, dim=128, rot=64,
             mode="interleaved", scaling="linear", factor=4.0, start=0, dtype="bf16"),
        # The gradient of the rotation in fp32, the precision the reference computes in.
        dict(name="rope_grad_f32", kind="rope", dir="bwd", batch=4, seq=1000, heads=24, dim=64, rot=64, mode="half",
             scaling="ntk", factor=2.0, start=0, dtype="f32"),
        # One new token for each of 64 running sequences, grouped key heads.
        dict(name="qk_token", kind="qk", dir="fwd", batch=64, seq=1, qh=16, kh=4, dim=128, rot=128, mode="half",
             start=4000, dtype="bf16"),
        # Two long prompts: from the fused projection's rows to the attention's head-first q, k, v.
        dict(name="qk_prompt", kind="qk", dir="fwd", batch=2, seq=8192, qh=32, kh=8, dim=128, rot=128, mode="half",
             start=0, dtype="bf16"),
        # A training batch: forward and backward, with the gradients of both norms' weights.
        dict(name="qk_train", kind="qk", dir="both", batch=4, seq=4096, qh=32, kh=8, dim=128, rot=128, mode="half",
             start=0, dtype="bf16"),
        # The backward alone in fp32, odd length, a head size no power of two, half of it rotated.
        dict(name="qk_grad_f32", kind="qk", dir="bwd", batch=3, seq=777, qh=8, kh=2, dim=96, rot=48, mode="interleaved",
             start=0, dtype="f32"),
        # Scores of a few tokens under the model: the head's weights are read once for 16 rows.
        dict(name="xent_few", kind="xent", dir="fwd", tokens=16, d=2048, vocab=32000, dtype="bf16", de="f32"),
        # The repository's decoder: its head's loss and gradients over a ragged batch, fp32 weight gradient.
        dict(name="xent_decoder", kind="xent", dir="both", tokens=8190, d=768, vocab=32000, dtype="bf16", de="f32"),
        # A vocabulary that no tile divides, the weight gradient kept in bf16.
        dict(name="xent_odd", kind="xent", dir="both", tokens=2001, d=1024, vocab=50001, dtype="bf16", de="bf16"),
        # The fp32 head at a ragged batch.
        dict(name="xent_f32", kind="xent", dir="both", tokens=1003, d=768, vocab=32000, dtype="f32", de="f32"),
        # A large vocabulary over a large batch: its logits would be 4 GB in fp32.
        dict(name="xent_large", kind="xent", dir="both", tokens=8192, d=2048, vocab=128000, dtype="bf16", de="f32"),
    ]


# ---- ranges --------------------------------------------------------------------------------
def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "qk", "qk", "xent", "xent"])
    if kind == "xent":
        # vocabularies odd as often as not; widths are multiples of 8 or, now and then, of 2
        d = 8 * _log(rng, 8, 256) if rng.random() < 0.85 else 2 * _log(rng, 32, 500)
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        tokens = _log(rng, 1, 8192 if dtype == "bf16" else 2048)
        return dict(kind=kind, dir=rng.choice(["fwd", "both", "both"]), tokens=tokens, d=d,
                    vocab=_log(rng, 500, 128000 if dtype == "bf16" else 50000), dtype=dtype,
                    de=rng.choice(["f32", "bf16"]) if dtype == "bf16" else "f32")
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
    mode = rng.choice(["half", "interleaved"])
    seq = 1 if rng.random() < 0.3 else _log(rng, 2, 16384)
    batch = max(1, min(_log(rng, 1, 128), 16384 // seq))
    start = rng.choice([0, rng.randint(1, 1000000)])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "rope":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(kind=kind, dir=rng.choice(["fwd", "bwd"]), batch=batch, seq=seq, heads=rng.randint(1, 40), dim=dim,
                    rot=rot, mode=mode, scaling=scaling, factor=1.0 if scaling == "none" else float(2 ** rng.randint(1, 5)),
                    start=start, dtype=dtype)
    kh = rng.randint(1, 8)
    return dict(kind=kind, dir=rng.choice(["fwd", "bwd", "both"]), batch=batch, seq=seq, qh=kh * rng.randint(1, 4), kh=kh,
                dim=dim, rot=rot, mode=mode, start=start, dtype=dtype)


# ---- inputs --------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype).contiguous()


def _freqs(rot, scaling, factor):
    """Angle of one position step of each pair in fp64, and the factor on cos and sin: theta 10000,
    plain, positions divided (linear), a larger base (ntk), or a ramp between the plain and the divided
    frequencies by how often a pair turns within the 4096 positions trained on (yarn)."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    theta = 10000.0
    if scaling == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2.0))
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = 4096.0 * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f.to(DEV), 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return {"rope": _prepare_rope, "qk": _prepare_qk, "xent": _prepare_xent}[case["kind"]](case, g)


def _positions(case, g):
    """int32 [batch, seq]: sequences that have got differently far."""
    B, S = case["batch"], case["seq"]
    first = case["start"] + torch.randint(0, 1000, (B, 1), device=DEV, generator=g)
    return (first + torch.arange(S, device=DEV)).to(torch.int32).contiguous()


def _prepare_rope(case, g):
    B, S, H, D = case["batch"], case["seq"], case["heads"], case["dim"]
    f, m = _freqs(case["rot"], case["scaling"], case["factor"])
    std = 0.01 if case["dir"] == "bwd" else 1.0
    return dict(case=case, x=_randn(g, B, S, H, D, std=std, dtype=TYPES[case["dtype"]]), pos=_positions(case, g), f=f, m=m)


def _prepare_qk(case, g):
    B, S, Q, K, D = case["batch"], case["seq"], case["qh"], case["kh"], case["dim"]
    dt = TYPES[case["dtype"]]
    s = dict(case=case, qkv=_randn(g, B, S, (Q + 2 * K) * D, dtype=dt), wq=1 + _randn(g, D, std=0.1, dtype=dt),
             wk=1 + _randn(g, D, std=0.1, dtype=dt), pos=_positions(case, g), f=_freqs(case["rot"], "none", 1.0)[0])
    if case["dir"] != "fwd":
        s.update(dq=_randn(g, B, Q, S, D, std=0.01, dtype=dt), dk=_randn(g, B, K, S, D, std=0.01, dtype=dt),
                 dv=_randn(g, B, K, S, D, std=0.01, dtype=dt))
    return s


def _prepare_xent(case, g):
    T, d, V = case["tokens"], case["d"], case["vocab"]
    dt = TYPES[case["dtype"]]
    E = _randn(g, V, d, std=0.02, dtype=dt)
    # frequent and rare tokens; a row leans towards its target by between nothing and much
    t = (V * torch.rand(T, device=DEV, generator=g) ** 3).long().clamp(0, V - 1)
    lean = 12.0 * torch.rand(T, 1, device=DEV, generator=g) / (0.02 ** 2 * d)
    h = (torch.randn(T, d, device=DEV, generator=g) + lean * E[t].float()).to(dt).contiguous()
    # one row in ten belongs to a prompt or to padding and has no target
    t = torch.where(torch.rand(T, device=DEV, generator=g) < 0.1, torch.full_like(t, -100), t)
    n = (t >= 0).sum().clamp(min=1)
    return dict(case=case, h=h, E=E, t=t.to(torch.int32).contiguous(),
                u=(torch.ones(T, device=DEV) / n).contiguous())


# ---- one pass ------------------------------------------------------------------------------
def run(s):
    return {"rope": _run_rope, "qk": _run_qk, "xent": _run_xent}[s["case"]["kind"]](s)


def _run_rope(s):
    c = s["case"]
    if own:
        import gn_bwd as gn
        call = gn.rope_fwd if c["dir"] == "fwd" else gn.rope_bwd
        return call(s["x"], s["f"], mode=c["mode"], positions=s["pos"], mscale=s["m"])
    cos, sin = _cos_sin(s["pos"], s["f"], s["m"])
    return _rotate(s["x"].float(), cos, sin if c["dir"] == "fwd" else -sin, c["rot"], c["mode"]).to(s["x"].dtype)


def _cos_sin(pos, f, m):
    """fp32 [batch, seq, 1, rot/2]; the angles of far positions need 64 bits."""
    a = pos.double()[:, :, None, None] * f
    return (torch.cos(a) * m).float(), (torch.sin(a) * m).float()


def _rotate(x, cos, sin, rot, mode):
    if mode == "interleaved":
        u, w = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        u, w = x[..., :rot // 2], x[..., rot // 2:rot]
    a, b = u * cos - w * sin, w * cos + u * sin
    r = torch.stack((a, b), -1).flatten(-2) if mode == "interleaved" else torch.cat((a, b), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _split(s):
    """q, k, v [batch, seq, heads, dim]: views of the fused projection's rows."""
    c = s["case"]
    B, S, Q, K, D = c["batch"], c["seq"], c["qh"], c["kh"], c["dim"]
    x = s["qkv"].view(B, S, Q + 2 * K, D)
    return x[:, :, :Q], x[:, :, Q:Q + K], x[:, :, Q + K:]


def _run_qk(s):
    c = s["case"]
    q, k, v = _split(s)
    out = {}
    if own:
        import gn_bwd as gn
        kw = dict(mode=c["mode"], positions=s["pos"], eps=1e-6, heads_first=True)
        if c["dir"] != "bwd":
            out["q"], out["k"], out["v"] = gn.qk_norm_rope_fwd(q, k, s["wq"], s["wk"], s["f"], v=v, **kw)
        if c["dir"] != "fwd":
            dqkv = torch.empty_like(s["qkv"])
            dq, dk, dv = _split(dict(case=c, qkv=dqkv))
            g = gn.qk_norm_rope_bwd(s["dq"], s["dk"], q, k, s["wq"], s["wk"], s["f"], dyv=s["dv"], out=(dq, dk, dv), **kw)
            out["dwq"], out["dwk"], out["dqkv"] = g[-2], g[-1], dqkv
        return out
    cos, sin = _cos_sin(s["pos"], s["f"], 1.0)
    if c["dir"] != "bwd":
        out["q"], out["k"] = _norm_rope(q, s["wq"], cos, sin, c), _norm_rope(k, s["wk"], cos, sin, c)
        out["v"] = v.transpose(1, 2).contiguous()
    if c["dir"] != "fwd":
        dq, out["dwq"] = _norm_rope_grad(q, s["wq"], s["dq"], cos, sin, c)
        dk, out["dwk"] = _norm_rope_grad(k, s["wk"], s["dk"], cos, sin, c)
        out["dqkv"] = torch.cat((dq, dk, s["dv"].transpose(1, 2)), 2).flatten(2)
    return out


def _norm_rope(x, w, cos, sin, c):
    f = x.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * w.float()
    return _rotate(n, cos, sin, c["rot"], c["mode"]).to(x.dtype).transpose(1, 2).contiguous()


def _norm_rope_grad(x, w, dy, cos, sin, c):
    f, w = x.float(), w.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
    g = _rotate(dy.transpose(1, 2).float(), cos, -sin, c["rot"], c["mode"])
    wg = w * g
    dx = r * (wg - f * (r * r) * (wg * f).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * f * r).sum((0, 1, 2), dtype=torch.float64).float()


def _run_xent(s):
    c = s["case"]
    h, E, t = s["h"], s["E"], s["t"]
    if own:
        import gn_bwd as gn
        loss, lse = gn.linear_xent_fwd(h, E, t)
        if c["dir"] == "fwd":
            return dict(loss=loss, lse=lse)
        dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=s["u"], dE_dtype=TYPES[c["de"]])
        return dict(loss=loss, lse=lse, dh=dh, dE=dE)
    hf, Ef = h.float(), E.float()
    l = hf @ Ef.t()
    m = l.max(-1, keepdim=True).values
    e = torch.exp(l - m)
    z = e.sum(-1, keepdim=True, dtype=torch.float64)
    lse = (m + torch.log(z))[:, 0]
    keep, at = t >= 0, t.long().clamp(min=0)
    rows = torch.arange(len(t), device=t.device)
    loss = torch.where(keep, lse - l[rows, at], 0.0).float()
    if c["dir"] == "fwd":
        return dict(loss=loss, lse=lse.float())
    del l
    G = e / z.float()
    G[rows, at] -= 1.0
    G *= torch.where(keep, s["u"], 0.0)[:, None]
    return dict(loss=loss, lse=lse.float(), dh=(G @ Ef).to(h.dtype), dE=(G.t() @ hf).to(TYPES[c["de"]]))


# ---- what a pass cannot do without -----------------------------------------------------------
def work(c):
    e = BYTES[c["dtype"]]
    if c["kind"] == "rope":
        n = c["batch"] * c["seq"] * c["heads"] * c["dim"]
        return dict(bytes=2 * n * e + 4 * c["batch"] * c["seq"] + 4 * c["rot"], flops=3 * n * c["rot"] // c["dim"])
    if c["kind"] == "qk":
        tok, D = c["batch"] * c["seq"], c["dim"]
        qk, v = tok * (c["qh"] + c["kh"]) * D, tok * c["kh"] * D
        b, f = 4 * tok + 4 * c["rot"] + 2 * D * e, 0
        if c["dir"] != "bwd":
            b, f = b + 2 * (qk + v) * e, f + 8 * qk
        if c["dir"] != "fwd":
            # the same q and k are read once for both directions
            b, f = b + (2 * qk + 2 * v + (qk if c["dir"] == "bwd" else 0)) * e + 8 * D, f + 16 * qk
        return dict(bytes=b, flops=f)
    T, d, V = c["tokens"], c["d"], c["vocab"]
    b, f = (T + V) * d * e + 12 * T, 2 * T * d * V
    if c["dir"] == "both":
        b, f = b + T * d * e + V * d * BYTES[c["de"]] + 4 * T, 3 * f
    return dict(bytes=b, flops=f)


# ---- the same in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"rope": _exact_rope, "qk": _exact_qk, "xent": _exact_xent}[case["kind"]](s)


def _turn(x, pos, f, m, rot, mode):
    """The rotation as a product of complex numbers."""
    by = torch.polar(torch.full((), m, dtype=torch.float64, device=x.device).expand(*pos.shape, 1, len(f)),
                     (pos.double()[..., None] * f)[:, :, None])
    part = x[..., :rot]
    if mode == "interleaved":
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2)) * by
        r = torch.view_as_real(z).reshape(part.shape)
    else:
        z = torch.complex(*part.chunk(2, -1)) * by
        r = torch.cat((z.real, z.imag), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _exact_rope(s):
    c = s["case"]
    x = s["x"].double()
    if c["dir"] == "fwd":
        return _turn(x, s["pos"], s["f"], s["m"], c["rot"], c["mode"])
    z = torch.zeros_like(x).requires_grad_()
    _turn(z, s["pos"], s["f"], s["m"], c["rot"], c["mode"]).backward(x)
    return z.grad


def _exact_qk(s):
    c = s["case"]
    qkv = s["qkv"].double().requires_grad_()
    wq, wk = s["wq"].double().requires_grad_(), s["wk"].double().requires_grad_()
    q, k, v = _split(dict(case=c, qkv=qkv))
    y = [_turn(x / ((x ** 2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * w, s["pos"], s["f"], 1.0, c["rot"],
               c["mode"]).permute(0, 2, 1, 3) for x, w in ((q, wq), (k, wk))] + [v.permute(0, 2, 1, 3)]
    out = {}
    if c["dir"] != "bwd":
        out.update(q=y[0].detach().contiguous(), k=y[1].detach().contiguous(), v=y[2].detach().contiguous())
    if c["dir"] != "fwd":
        torch.autograd.backward(y, [s["dq"].double(), s["dk"].double(), s["dv"].double()])
        out.update(dqkv=qkv.grad, dwq=wq.grad, dwk=wk.grad)
    return out


def _exact_xent(s):
    c = s["case"]
    h, E, t = s["h"].double(), s["E"].double(), s["t"].long()
    logp = h @ E.t()
    lse = torch.logsumexp(logp, -1)
    logp -= lse[:, None]
    valid = t >= 0
    hit = torch.nonzero(valid)[:, 0]
    loss = torch.zeros_like(lse)
    loss[hit] = -logp[hit, t[hit]]
    if c["dir"] == "fwd":
        return dict(loss=loss, lse=lse)
    u = s["u"].double() * valid
    G = logp.exp_().mul_(u[:, None])
    G[hit, t[hit]] -= u[hit]
    return dict(loss=loss, lse=lse, dh=G @ E, dE=G.t() @ h)
