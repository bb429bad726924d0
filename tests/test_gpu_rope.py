"""GPU tests of rotary positions (rope) and per-head query/key norms with the rotation
(qk_norm_rope), against plain fp64 torch: layouts, partial rotation, positions, strides, single
tokens, odd lengths, gradients, in-place use, streams, graph replays.

Tolerances, element by element.  Rounding to the output type: half a step, finfo.eps / 2 of the
value.  Before it, in fp32: the angle in turns is rounded to 2^-26, which moves cos and sin by
2 pi 2^-26 < 2 * 2^-24; they are good to 2 steps, 2 * 2^-23; products and their sum add three half
steps: together below 2^-20 (|u| + |w|) of a pair.  The norm's sum of squares has at most D / 2 + 6
roundings in a chain (D <= 512, but 16 to 22 in practice) and the reciprocal root one: r within
2^-17.  A gradient adds the mean of w g x, likewise, so 2^-16 of the sum of its terms' magnitudes."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DEV = "cuda:0"


@pytest.fixture(scope="module")
def gn(gpu):
    import gn_bwd
    gn_bwd.lib()
    return gn_bwd


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def rand(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def turn(x, pos, f, m, mode, back=False):
    """x [B, S, H, D] fp64 rotated by pos [B, S]."""
    rot = 2 * len(f)
    a = pos.double()[:, :, None, None] * f
    c, s = m * torch.cos(a), (-m if back else m) * torch.sin(a)
    y = x.clone()
    u, w = (slice(0, rot, 2), slice(1, rot, 2)) if mode == "interleaved" else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., u] = x[..., u] * c - x[..., w] * s
    y[..., w] = x[..., w] * c + x[..., u] * s
    return y


def near(got, ref, size):
    """|got - ref| <= its type's rounding of ref + 'size'."""
    e = torch.finfo(got.dtype).eps / 2
    d = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    bad = d > e * ref.abs() + size + torch.finfo(got.dtype).tiny
    assert not bool(bad.any()), (float((d / (e * ref.abs() + size + 1e-300)).max()), int(bad.sum()))


def row_max(x):
    return x.abs().amax(-1, keepdim=True)


def freqs(rot, theta=10000.0):
    return (theta ** (-torch.arange(rot // 2, dtype=F64, device=DEV) * 2 / max(rot, 1)))


SHAPES = [  # B, S, H, D, rot
    (1, 1, 1, 2, 2), (1, 1, 3, 64, 64), (2, 5, 3, 32, 32), (3, 7, 5, 64, 32), (2, 33, 4, 128, 128),
    (1, 129, 2, 96, 48), (2, 9, 3, 80, 80), (2, 9, 3, 80, 26), (1, 17, 2, 256, 256), (1, 5, 1, 512, 512),
    (5, 1, 12, 128, 64), (1, 3, 7, 40, 20), (1, 2500, 3, 64, 64), (2, 3, 2, 192, 192), (1, 11, 1, 510, 34),
    (1, 3, 40, 16, 16), (1, 4, 2, 48, 0)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("mode", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,H,D,rot", SHAPES)
def test_rope(gn, B, S, H, D, rot, mode, dtype):
    g = gen(B + S + H + D)
    x = rand(g, B, S, H, D, dtype=dtype)
    pos = torch.randint(0, 5000, (B, S), device=DEV, generator=g).to(torch.int32)
    f = freqs(rot)
    y = gn.rope_fwd(x, f, mode=mode, positions=pos, mscale=1.25)
    near(y, turn(x.double(), pos, f, 1.25, mode), 2.0 ** -20 * 2.5 * row_max(x.double()))
    dx = gn.rope_bwd(x, f, mode=mode, positions=pos, mscale=1.25)
    near(dx, turn(x.double(), pos, f, 1.25, mode, back=True), 2.0 ** -20 * 2.5 * row_max(x.double()))
    # positions counted from pos0
    y0 = gn.rope_fwd(x, f, mode=mode, pos0=70)
    p0 = (70 + torch.arange(S, device=DEV))[None].expand(B, S)
    near(y0, turn(x.double(), p0, f, 1.0, mode), 2.0 ** -20 * 2 * row_max(x.double()))
    p1 = p0[0].to(torch.int32).contiguous()
    assert torch.equal(y0, gn.rope_fwd(x, f, mode=mode, positions=p1))


@pytest.mark.parametrize("first", [0, 2 ** 20, 2 ** 31 - 1, -(2 ** 31)])
def test_rope_far_positions(gn, first):
    """Angles of far positions are formed in 64 bits."""
    x = rand(gen(3), 1, 1, 2, 64, dtype=F32)
    f = freqs(64)
    pos = torch.tensor([[first]], dtype=torch.int32, device=DEV)
    # the reference's own angle: 2^31 radians in fp64 are good to 2^-21
    near(gn.rope_fwd(x, f, positions=pos), turn(x.double(), pos, f, 1.0, "half"), 2.0 ** -19 * 2 * row_max(x.double()))


@pytest.mark.parametrize("pos0", [2 ** 31 - 1, -(2 ** 31)])
def test_rope_far_first_position(gn, pos0):
    """A first position at the border of 32 bits counts on past it."""
    x = rand(gen(4), 1, 3, 2, 64, dtype=F32)
    f = freqs(64)
    pos = pos0 + torch.arange(3, dtype=torch.int64, device=DEV)[None]
    near(gn.rope_fwd(x, f, pos0=pos0), turn(x.double(), pos, f, 1.0, "half"), 2.0 ** -19 * 2 * row_max(x.double()))


@pytest.mark.parametrize("mode", ["half", "interleaved"])
def test_rope_views(gn, mode):
    """Heads of fused rows, head-first tensors, unaligned and broadcast views, in-place use; what
    lies between the heads stays as it was."""
    g = gen(11)
    B, S, H, D = 2, 37, 3, 64
    f = freqs(D)
    fused = rand(g, B, S, 2 * H + 1, D)
    keep = fused.clone()
    x = fused[:, :, 1:1 + H]
    ref = turn(x.double(), torch.arange(S, device=DEV)[None].expand(B, S), f, 1.0, mode)
    size = 2.0 ** -20 * 2 * row_max(x.double())
    y = gn.rope_fwd(x, f, mode=mode)
    near(y, ref, size)
    hf = torch.zeros(B, H, S, D, device=DEV, dtype=BF)
    assert gn.rope_fwd(x, f, mode=mode, out=hf.transpose(1, 2)) is not None
    assert torch.equal(hf.transpose(1, 2), y)
    odd = torch.full((B * S * H * D + 1,), 7.0, device=DEV, dtype=BF)
    gn.rope_fwd(x, f, mode=mode, out=odd[1:].view(B, S, H, D))  # element by element
    near(odd[1:].view(B, S, H, D), ref, size)
    assert float(odd[0]) == 7.0
    one = x[:, :1].expand(B, S, H, D)  # the same token at every position
    near(gn.rope_fwd(one, f, mode=mode), turn(one.double(), torch.arange(S, device=DEV)[None].expand(B, S), f, 1.0, mode),
         2.0 ** -20 * 2 * row_max(one.double()))
    gn.rope_fwd(x, f, mode=mode, out=x)
    assert torch.equal(x, y)
    assert torch.equal(fused[:, :, :1], keep[:, :, :1]) and torch.equal(fused[:, :, 1 + H:], keep[:, :, 1 + H:])


def test_rope_empty(gn):
    f = freqs(64)
    assert gn.rope_fwd(torch.empty(0, 4, 2, 64, device=DEV, dtype=BF), f).shape == (0, 4, 2, 64)
    assert gn.rope_fwd(torch.empty(2, 0, 2, 64, device=DEV, dtype=BF), f).shape == (2, 0, 2, 64)
    assert gn.rope_fwd(torch.empty(2, 4, 0, 64, device=DEV, dtype=BF), f).shape == (2, 4, 0, 64)


def test_rope_large_offsets(gn):
    """A head-first tensor whose last elements lie past 2^31 elements."""
    B, S, H, D = 1, 2 ** 18 + 3, 130, 64
    big = torch.empty(B, H, S, D, device=DEV, dtype=BF)
    assert big.numel() > 2 ** 31
    part = big[:, :, -5:].transpose(1, 2)
    part.copy_(rand(gen(5), B, 5, H, D))
    ref = turn(part.double(), (9 + torch.arange(5, device=DEV))[None], freqs(D), 1.0, "half")
    size = 2.0 ** -20 * 2 * row_max(part.double())
    gn.rope_fwd(part, freqs(D), pos0=9, out=part)
    near(part, ref, size)


# ---- norms with the rotation ------------------------------------------------------------------
def normed(x, w, eps=1e-6):
    r = (x.double().square().mean(-1, keepdim=True) + eps).rsqrt()
    return x.double() * r * (1.0 if w is None else w.double())


def grads(x, w, dy, pos, f, m, mode, eps=1e-6):
    """dx, dw and the magnitudes of their terms, from the formulas, fp64."""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], device=DEV, dtype=F64) if w is None else w.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = dy if f is None else turn(dy, pos, f, m, mode, back=True)
    dx = r * (w * g - x * r * r * (w * g * x).mean(-1, keepdim=True))
    # the rotation's rounding is relative to its pair: to the row's largest element
    gm = row_max(dy) * 2 * abs(m) + 0 * dy
    size = r * (w.abs() * gm + x.abs() * r * r * (w.abs() * gm * x.abs()).mean(-1, keepdim=True))
    return dx, (g * x * r).sum((0, 1, 2)), size, (gm * x.abs() * r).sum((0, 1, 2))


QK = [  # B, S, Hq, Hk, D, rot
    (1, 1, 1, 1, 64, 64), (4, 1, 8, 2, 128, 128), (2, 33, 4, 2, 64, 32), (3, 7, 6, 3, 96, 48), (1, 129, 3, 1, 80, 10),
    (2, 5, 2, 2, 256, 256), (1, 600, 4, 4, 32, 32), (1, 3, 2, 1, 34, 34), (1, 2100, 2, 1, 64, 0), (1, 5, 1, 1, 512, 512)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("mode", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,Hq,Hk,D,rot", QK)
def test_qk_norm_rope(gn, B, S, Hq, Hk, D, rot, mode, dtype):
    g = gen(B + S + Hq + D)
    qkv = rand(g, B, S, Hq + 2 * Hk, D, dtype=dtype)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    wq, wk = rand(g, D, dtype=dtype), rand(g, D, dtype=dtype)
    pos = torch.randint(0, 3000, (B, S), device=DEV, generator=g).to(torch.int32)
    f = freqs(rot) if rot else None
    kw = dict(mode=mode, positions=pos, mscale=0.75 if rot else 1.0)
    m = kw["mscale"]
    yq, yk, yv = gn.qk_norm_rope_fwd(q, k, wq, wk, f, v=v, heads_first=True, **kw)
    for y, x, w in ((yq, q, wq), (yk, k, wk)):
        n = normed(x, w)
        ref = n if f is None else turn(n, pos, f, m, mode)
        near(y.transpose(1, 2), ref, 2.0 ** -16 * 2 * row_max(n))
    assert torch.equal(yv.transpose(1, 2), v)
    yq2, yk2 = gn.qk_norm_rope_fwd(q, k, wq, wk, f, **kw)
    assert torch.equal(yq2, yq.transpose(1, 2)) and torch.equal(yk2, yk.transpose(1, 2))

    dyq, dyk, dyv = (rand(g, B, H, S, D, dtype=dtype) for H in (Hq, Hk, Hk))
    dqkv = torch.full_like(qkv, float("nan"))
    out = (dqkv[:, :, :Hq], dqkv[:, :, Hq:Hq + Hk], dqkv[:, :, Hq + Hk:])
    got = gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f, dyv=dyv, heads_first=True, out=out, **kw)
    assert torch.equal(out[2], dyv.transpose(1, 2))
    # dw: a lane's chain is its rows, then the lane groups, then the blocks
    chain = (B * S * max(Hq, Hk) // 4 + 400) * 2.0 ** -24
    for dx, dw, x, w, dy in ((out[0], got[3], q, wq, dyq), (out[1], got[4], k, wk, dyk)):
        ref, rw, size, sw = grads(x, w, dy.transpose(1, 2), pos, f, m, mode)
        near(dx, ref, 2.0 ** -16 * size)
        assert bool(((dw.double() - rw).abs() <= (2.0 ** -16 + chain) * sw).all())
    again = gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f, heads_first=True, **kw)
    assert again[2] is None and torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    assert torch.equal(again[3], got[3]) and torch.equal(again[4], got[4])
    one = torch.ones(D, device=DEV)
    gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f, heads_first=True, dwq=one, dwk=one.clone(), accumulate=True, **kw)
    assert torch.equal(one, got[3] + 1)


def test_qk_interleaved_heads_in_place(gn):
    """q, k and v of a head side by side ([B, S, H, 3, D]), normed where they lie, and their gradients
    in one tensor of that layout."""
    g = gen(21)
    B, S, H, D = 2, 19, 4, 64
    x, dy = rand(g, B, S, H, 3, D), rand(g, B, S, H, 3, D)
    w, f = rand(g, D), freqs(D)
    a, b = gn.qk_norm_rope_fwd(x[:, :, :, 0].contiguous(), x[:, :, :, 1].contiguous(), w, w, f)
    dq, dk, _, dwq, dwk = gn.qk_norm_rope_bwd(dy[:, :, :, 0].contiguous(), dy[:, :, :, 1].contiguous(), x[:, :, :, 0], x[:, :, :, 1],
                                              w, w, f)
    dx = torch.zeros_like(x)
    got = gn.qk_norm_rope_bwd(dy[:, :, :, 0], dy[:, :, :, 1], x[:, :, :, 0], x[:, :, :, 1], w, w, f, dyv=dy[:, :, :, 2],
                              out=[dx[:, :, :, i] for i in range(3)])
    assert torch.equal(dx[:, :, :, 0], dq) and torch.equal(dx[:, :, :, 1], dk) and torch.equal(dx[:, :, :, 2], dy[:, :, :, 2])
    assert torch.equal(got[3], dwq) and torch.equal(got[4], dwk)
    keep = x.clone()
    parts = [x[:, :, :, i] for i in range(3)]
    gn.qk_norm_rope_fwd(*parts[:2], w, w, f, v=parts[2], out=parts)
    assert torch.equal(x[:, :, :, 0], a) and torch.equal(x[:, :, :, 1], b) and torch.equal(x[:, :, :, 2], keep[:, :, :, 2])


def test_qk_without_weights_keys_or_dw(gn):
    g = gen(2)
    q, dy = rand(g, 2, 9, 3, 64), rand(g, 2, 9, 3, 64)
    f = freqs(64)
    pos = torch.arange(9, device=DEV)[None].expand(2, 9)
    yq, yk = gn.qk_norm_rope_fwd(q, None, freqs=f)
    assert yk is None
    n = normed(q, None)
    near(yq, turn(n, pos, f, 1.0, "half"), 2.0 ** -15 * row_max(n))
    dq, dk, dv, dwq, dwk = gn.qk_norm_rope_bwd(dy, None, q, None, freqs=f, need_dw=False)
    assert dk is None and dv is None and dwq is None and dwk is None
    ref, rw, size, sw = grads(q, None, dy, pos, f, 1.0, "half")
    near(dq, ref, 2.0 ** -16 * size)
    dwq = gn.qk_norm_rope_bwd(dy, None, q, None, freqs=f)[3]
    assert bool(((dwq.double() - rw).abs() <= 2.0 ** -15 * sw).all())


def test_qk_gradient_against_differences(gn):
    """fp32, a central difference along a random direction of q, k and both weights."""
    g = gen(8)
    B, S, Hq, Hk, D = 1, 6, 2, 1, 32
    q, k, wq, wk = (rand(g, *s, dtype=F32) for s in ((B, S, Hq, D), (B, S, Hk, D), (D,), (D,)))
    dyq, dyk = rand(g, B, S, Hq, D, dtype=F32), rand(g, B, S, Hk, D, dtype=F32)
    f = freqs(16)

    def value(q, k, wq, wk):
        yq, yk = gn.qk_norm_rope_fwd(q, k, wq, wk, f)
        return float((yq.double() * dyq).sum() + (yk.double() * dyk).sum())

    dq, dk, _, dwq, dwk = gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f)
    args, ds = (q, k, wq, wk), (dq, dk, dwq, dwk)
    t = [rand(g, *a.shape, dtype=F32) for a in args]
    h = 2.0 ** -6
    slope = (value(*(a + h * b for a, b in zip(args, t))) - value(*(a - h * b for a, b in zip(args, t)))) / (2 * h)
    want = sum(float((a.double() * b).sum()) for a, b in zip(ds, t))
    # the values' fp32 error (2^-16 of ~600 terms of size 1, over h) and the third difference
    assert abs(slope - want) <= 600 * 2.0 ** -16 / h * 0.1 + 0.02 * sum(float((a * b).abs().sum()) for a, b in zip(ds, t))


def test_zero_rows_and_padding(gn):
    """Rows of zeros (padding) give zeros and finite gradients, and rows with inf or NaN stay alone."""
    g = gen(4)
    q = rand(g, 1, 8, 2, 64)
    q[0, 2] = 0
    q[0, 5] = float("nan")
    q[0, 6, 0, 3] = float("inf")
    f = freqs(64)
    y, _ = gn.qk_norm_rope_fwd(q, None, freqs=f)
    assert bool((y[0, 2] == 0).all())
    clean = [0, 1, 2, 3, 4, 7]
    assert bool(torch.isfinite(y[0, clean]).all()) and bool(torch.isfinite(y[0, 6, 1]).all())
    assert bool(torch.isnan(y[0, 5]).all())
    dq = gn.qk_norm_rope_bwd(torch.ones_like(q), None, q, None, freqs=f, need_dw=False)[0]
    assert bool(torch.isfinite(dq[0, clean]).all())


def test_qk_empty(gn):
    e = torch.empty(2, 0, 3, 64, device=DEV, dtype=BF)
    one = torch.ones(64, device=DEV)
    out = gn.qk_norm_rope_bwd(e, e, e, e, dwq=one, dwk=one.clone(), freqs=freqs(64))
    assert bool((out[3] == 0).all()) and bool((out[4] == 0).all())
    one.fill_(1)
    out = gn.qk_norm_rope_bwd(e, e, e, e, dwq=one, dwk=one.clone(), freqs=freqs(64), accumulate=True)
    assert bool((out[3] == 1).all())


def test_qk_on_another_stream_and_replayed(gn):
    """On a side stream, and captured forward and backward replayed with new inputs between eager work."""
    g = gen(6)
    B, S, Hq, Hk, D = 2, 300, 4, 2, 128
    q, k = rand(g, B, S, Hq, D), rand(g, B, S, Hk, D)
    wq, wk, f = rand(g, D), rand(g, D), freqs(D)

    def both(ws):
        yq, yk = gn.qk_norm_rope_fwd(q, k, wq, wk, f)
        return (yq, yk, *gn.qk_norm_rope_bwd(yq, yk, q, k, wq, wk, f, ws=ws))

    ws = gn.workspace(gn.qk_norm_rope_workspace_bytes(B, S, D), DEV)
    eager = both(ws)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = both(gn.workspace(gn.qk_norm_rope_workspace_bytes(B, S, D), DEV))
    s.synchronize()
    for a, b in zip(eager, other):
        assert a is b or torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(ws)
    for i in range(3):
        q.copy_(rand(gen(20 + i), B, S, Hq, D))
        k.copy_(rand(gen(30 + i), B, S, Hk, D))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(both(None), held):
            assert a is b or torch.equal(a, b)
