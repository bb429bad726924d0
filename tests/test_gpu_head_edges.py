"""GPU tests of the borders of rope, qk_norm_rope and linear_xent: a zero eps, infinities beside
elements that pass through, confident rows, launches past a dimension's limit, chained nodes.

Tolerances are those of test_gpu_rope.py and test_gpu_linear_xent.py where nothing else is said."""
import pytest

from test_gpu_rope import freqs, gen, grads, near, rand, row_max, turn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DEV = "cuda:0"


@pytest.fixture(scope="module")
def gn(gpu):
    import gn_bwd
    gn_bwd.lib()
    return gn_bwd


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("mode", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,Hq,Hk,D,rot", [(1, 1, 8, 2, 128, 128), (3, 7, 5, 1, 64, 32), (2, 9, 3, 1, 80, 26),
                                             (1, 1, 1, 1, 34, 0), (1, 2100, 3, 3, 96, 48)])
def test_norms_without_eps(gn, B, S, Hq, Hk, D, rot, mode, dtype):
    """eps = 0 over rows that are not zero, in tiles whose rows do not fill the block."""
    g = gen(B + S + D)
    q, k = rand(g, B, S, Hq, D, dtype=dtype), rand(g, B, S, Hk, D, dtype=dtype)
    dyq, dyk = rand(g, B, S, Hq, D, dtype=dtype), rand(g, B, S, Hk, D, dtype=dtype)
    wq, wk = rand(g, D, dtype=dtype), rand(g, D, dtype=dtype)
    f = freqs(rot) if rot else None
    pos = torch.arange(S, device=DEV)[None].expand(B, S)
    y = gn.qk_norm_rope_fwd(q, k, wq, wk, f, mode=mode, eps=0.0)
    dq, dk, _, dwq, dwk = gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f, mode=mode, eps=0.0)
    chain = (B * S * max(Hq, Hk) // 4 + 400) * 2.0 ** -24
    for x, w, dy, got, dx, dw in ((q, wq, dyq, y[0], dq, dwq), (k, wk, dyk, y[1], dk, dwk)):
        n = x.double() * x.double().square().mean(-1, keepdim=True).rsqrt() * w.double()
        near(got, n if f is None else turn(n, pos, f, 1.0, mode), 2.0 ** -16 * 2 * row_max(n))
        ref, rw, size, sw = grads(x, w, dy, pos, f, 1.0, mode, eps=0.0)
        near(dx, ref, 2.0 ** -16 * size)
        assert bool(((dw.double() - rw).abs() <= (2.0 ** -16 + chain) * sw).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("mode", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(64, 32), (80, 26), (128, 0), (34, 2)])
def test_elements_behind_the_rotation_pass_as_they_are(gn, D, rot, mode, dtype):
    """Bit for bit, beside infinities, NaN and negative zeros too."""
    g = gen(D)
    x = rand(g, 2, 9, 3, D, dtype=dtype)
    x[0, :, :, rot::5] = float("inf")
    x[1, 2, :, rot + 1::7] = float("nan")
    x[1, 3, :, rot::2] = -0.0
    bits = torch.int16 if dtype is BF else torch.int32
    f = freqs(rot)
    for fn in (gn.rope_fwd, gn.rope_bwd):
        y = fn(x, f, mode=mode, pos0=3)
        assert torch.equal(y[..., rot:].contiguous().view(bits), x[..., rot:].contiguous().view(bits))
        assert bool(torch.isfinite(y[..., :rot]).all())
    # the norm of a row with an infinity: r = 0, so its finite elements become 0, and no neighbour NaN
    y, _ = gn.qk_norm_rope_fwd(x[:1], None, freqs=f, mode=mode)
    fine = torch.isfinite(x[:1])
    assert bool((y[fine] == 0).all()) and bool(torch.isnan(y[~fine]).all())


@pytest.mark.parametrize("tokens", [2 ** 24 + 5, 2 ** 22 + 1])
def test_more_tiles_than_a_dimension_launches(gn, tokens):
    """One token a tile, more than 2^32 threads: every token is reached (rotation, and the norm)."""
    g = gen(1)
    H, D = 17, 2  # 34 elements a token: element by element, a tile is one token
    x = torch.randn(1, tokens, H, D, device=DEV, dtype=BF, generator=g)
    f = freqs(D)
    y = torch.full_like(x, float("nan"))
    gn.rope_fwd(x, f, out=y)
    back = gn.rope_bwd(y, f)
    # two roundings to bf16 of a pair's elements
    size = (2.0 ** -7 + 2.0 ** -18) * row_max(x.float())
    assert bool(((back.float() - x.float()).abs() <= size).all())
    at = [0, 1, tokens // 2, tokens - 6, tokens - 5, tokens - 1]
    near(y[:, at], turn(x[:, at].double(), torch.tensor([at], device=DEV), f, 1.0, "half"),
         2.0 ** -20 * 2 * row_max(x[:, at].double()))
    y.fill_(float("nan"))
    gn.qk_norm_rope_fwd(x, None, freqs=f, out=(y, None))
    norm = y.float().square().mean(-1)
    # each element of a pair off by 2^-8 of it, the norm by 2^-7; eps 1e-6 against mean(x^2)
    fine = x.float().square().mean(-1) > 2e-4
    assert bool(((norm - 1).abs() <= 2.0 ** -7 + 2.0 ** -7)[fine].all()) and bool(torch.isfinite(norm).all())


def some_rows(gn, h, E, t, at):
    """Gradients of a loss over the rows `at` (none twice) alone, the same in fp64 from those rows, and lse."""
    T = h.shape[0]
    assert len(at) == len(at.unique())
    u = torch.zeros(T, device=DEV)
    u[at] = torch.rand(len(at), device=DEV, generator=gen(3)) + 0.5
    loss, lse = gn.linear_xent_fwd(h, E, t)
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u)
    x, Ed = h[at].double(), E.double()
    l = x @ Ed.t()
    p = torch.softmax(l, -1)
    G = p.clone()
    G[torch.arange(len(at)), t[at].long()] -= 1
    G *= u[at].double()[:, None]
    size = torch.logsumexp(l, -1), (x.abs() @ Ed.abs().t()).amax(-1)
    # p: the logits' error and 2^-20 (1 + |l| + |lse|); 2^-24 of each of d terms
    d = h.shape[1]
    dp = p * (2 * (d * 2.0 ** -24 + 2.0 ** -22) * size[1] + 2.0 ** -20 * (2 + 2 * l.abs().amax(-1) + size[0].abs()))[:, None]
    dG = u[at].double()[:, None] * (dp + 2.0 ** -22)
    return loss, lse, dh, dE, l, G, dG, x, Ed


def test_rows_past_a_dimension_of_blocks(gn):
    """fp32, more than 2^24 rows (a row a block): the last ones' loss and gradients, and a tail of the
    vocabulary."""
    g = gen(2)
    T, d, V = 2 ** 24 + 9, 4, 5
    h = torch.randn(T, d, device=DEV, generator=g)
    E = torch.randn(V, d, device=DEV, generator=g)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    at = torch.tensor([0, 5, 2 ** 22, 2 ** 24 - 1, T - 9, T - 1], device=DEV)
    loss, lse, dh, dE, l, G, dG, x, Ed = some_rows(gn, h, E, t, at)
    logits = h.double() @ Ed.t()
    ref = torch.logsumexp(logits, -1)
    # 4 terms a logit, and exp, sum and log
    assert bool(((lse.double() - ref).abs() <= 2.0 ** -20 * (2 + logits.abs().amax(-1))).all())
    ref = ref - logits.gather(1, t.long()[:, None])[:, 0]
    assert bool(((loss.double() - ref).abs() <= 2.0 ** -19 * (2 + logits.abs().amax(-1))).all())
    bound = dG @ Ed.abs() + 2.0 ** -21 * (G.abs() @ Ed.abs())
    assert bool(((dh[at].double() - G @ Ed).abs() <= bound).all())
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert bool((dh[rest] == 0).all())
    assert bool(((dE.double() - G.t() @ x).abs() <= dG.t() @ x.abs() + 2.0 ** -20 * (G.t().abs() @ x.abs())).all())


def test_h_past_32_bits(gn):
    """bf16, an h and a dh of more than 2^31 elements."""
    g = gen(5)
    T, d, V = 2 ** 21 + 37, 1032, 300
    h = torch.empty(T, d, device=DEV, dtype=BF)
    for i in range(0, T, 2 ** 18):
        h[i:i + 2 ** 18].normal_(0, 1, generator=g)
    E = rand(g, V, d, std=0.05)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    at = torch.tensor([0, 1, 2 ** 20, T - 300, T - 2, T - 1], device=DEV)
    loss, lse, dh, dE, l, G, dG, x, Ed = some_rows(gn, h, E, t, at)
    ref = torch.logsumexp(l, -1)
    el = d * 2.0 ** -24 * (x.abs() @ Ed.abs().t()).amax(-1) + 2.0 ** -20 * (1 + l.abs().amax(-1))
    assert bool(((lse[at].double() - ref).abs() <= el).all())
    ref = ref - l.gather(1, t[at].long()[:, None])[:, 0]
    assert bool(((loss[at].double() - ref).abs() <= 2 * el).all())
    ref = G @ Ed  # G in bf16 but at the target, dh's own rounding, and a sum of 300 terms
    assert bool(((dh[at].double() - ref).abs() <= (dG + (2.0 ** -8 + 2.0 ** -15) * G.abs()) @ Ed.abs() + 2.0 ** -8 * ref.abs()).all())
    ref = G.t() @ x  # two pieces of G
    assert bool(((dE.double() - ref).abs() <= (dG.t() + 2.0 ** -16 * G.t().abs()) @ x.abs()).all())
    assert bool((dh[2:2 ** 20] == 0).all()) and bool((dh[2 ** 20 + 1:T - 300] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d", [(3, 64), (20, 256), (70, 64), (300, 40), (4100, 64)])
@pytest.mark.parametrize("V", [1, 40])
def test_a_certain_row_has_no_gradient(gn, T, d, V, dtype):
    """The target's logit is 300 (exact in either type and in lse) and nothing beside it: p = 1, no loss
    and no gradient.  exp2's argument is off by half a step of 300 log2e at most before it is put right, its
    value by 2^-22."""
    h, E = torch.zeros(T, d, device=DEV, dtype=dtype), torch.zeros(V, d, device=DEV, dtype=dtype)
    h[:, 0], E[0, 0] = 256, 1.171875
    t = torch.zeros(T, device=DEV, dtype=torch.int32)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    assert bool((lse == 300).all()) and bool((loss.abs() <= 2.0 ** -22).all())
    dh, dE = gn.linear_xent_bwd(h, E, t, lse)
    # G <= 2^-22 at the target, times E and h (and summed over the rows)
    assert bool((dh.float().abs() <= 2.0 ** -22 * 1.171875).all())
    assert bool((dE.abs() <= 2.0 ** -22 * 256 * T).all())
    # a row twice as certain of two equal columns: p = 1/2 each
    if V > 1:
        E[V - 1] = E[0]
        l = torch.full((T,), 300.0, device=DEV, dtype=F64)
        loss, lse = gn.linear_xent_fwd(h, E, t)
        ref = l + torch.log(torch.tensor(2.0, dtype=F64))
        assert bool(((lse.double() - ref).abs() <= 2.0 ** -16).all())  # half a step of 300
        dh, dE = gn.linear_xent_bwd(h, E, t, torch.full_like(lse, 300.0))  # lse as it was: p = 1 each
        assert bool((dE[0].abs() <= 2.0 ** -22 * 256 * T).all())
        assert bool(((dE[V - 1] - h.float().sum(0)).abs() <= 2.0 ** -22 * 256 * T).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d,V", [(7, 64, 900), (16, 256, 3000), (70, 64, 900), (300, 64, 901), (1003, 72, 2000)])
def test_small_losses_of_far_logits(gn, T, d, V, dtype):
    """Logits of some hundreds, whole numbers and so exact, the target the largest or the next: the loss
    keeps what lse has to round away.  s is good to 2^-19 (V terms of 2^-22 joined a few dozen times), ln s
    to that and 2^-22, and the sum is rounded once."""
    g = gen(T + V)
    h = torch.randint(-8, 9, (T, d), device=DEV, generator=g).to(dtype)
    E = torch.randint(-4, 5, (V, d), device=DEV, generator=g).to(dtype)
    l = h.double() @ E.double().t()
    best = l.topk(2, -1)
    t = best.indices.gather(1, (torch.arange(T, device=DEV) % 3 == 0).long()[:, None])[:, 0].to(torch.int32)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    top = best.values[:, :1]
    ref = torch.logsumexp(l - top, -1) + top[:, 0] - l.gather(1, t.long()[:, None])[:, 0]
    assert float(lse.max()) > 200
    assert bool(((loss.double() - ref).abs() <= 2.0 ** -19 + 2.0 ** -22 + 2.0 ** -24 * ref).all())


# ---- nodes of the tape ------------------------------------------------------------------------
@pytest.fixture(scope="module")
def tape_env(gn):
    import grilly_bridge as gb
    import grilly_core
    dev = grilly_core.Device(0)
    gb.attach_torch_stream(dev)
    return grilly_core, gb, dev


def node_grads(tape_env, op, ins, outs, params, saved, up, wanted):
    """The gradients (as fp32 host tensors) of `wanted` [(tensor, dtype code or None)] after one node."""
    gc, gb, dev = tape_env
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(getattr(gc.OpType, op), ins, outs, params)
    tape.save_for_backward(n, saved)
    tape.backward(n, up.data_ptr())
    got = []
    for t, dt in wanted:
        gid = tape.get_grad_buffer(t.data_ptr())
        got.append(torch.from_numpy(gb.download(dev, gid, t.shape, gb.dtype_code(t) if dt is None else dt)))
    tape.end()
    return got


@pytest.mark.parametrize("eps,mscale", [(0.0, 1.0), (0.0, 0.0), (1e-6, 0.0), (1e-3, 2.0)])
def test_nodes_take_zeros_at_their_word(gn, tape_env, eps, mscale):
    """An eps or an mscale of 0 in a node's parameters is the forward's, not a default (rows whose mean square
    is about 1e-6, where an eps of 1e-6 halves the norm)."""
    gc, gb, dev = tape_env
    g = gen(8)
    B, S, H, K, D, rot = 1, 5, 3, 1, 64, 32
    C = (H + 2 * K) * D
    x, dy = rand(g, B, S, C, dtype=F32, std=1e-3), rand(g, B, S, C, dtype=F32)
    wq, wk, f = rand(g, D, dtype=F32), rand(g, D, dtype=F32), freqs(rot)
    part = lambda t: (t.view(B, S, -1, D)[:, :, :H], t.view(B, S, -1, D)[:, :, H:H + K], t.view(B, S, -1, D)[:, :, H + K:])
    y, want = torch.empty_like(x), torch.empty_like(x)
    gn.qk_norm_rope_fwd(*part(x)[:2], wq, wk, f, v=part(x)[2], out=part(y), eps=eps, mscale=mscale)
    direct = gn.qk_norm_rope_bwd(*part(dy)[:2], *part(x)[:2], wq, wk, f, dyv=part(dy)[2], out=part(want), eps=eps,
                                 mscale=mscale)
    got = node_grads(tape_env, "QkNormRope", [gb.tref(x, True)], [gb.tref(y)],
                     gb.qk_norm_rope_params(H, K, rot, eps=eps, mscale=mscale), [wq.data_ptr(), wk.data_ptr(), f.data_ptr()],
                     dy, [(x, None), (wq, gb.DTYPE_F32), (wk, gb.DTYPE_F32)])
    for a, b in zip(got, (want, direct[3], direct[4])):
        assert torch.equal(a, b.cpu()) and bool(torch.isfinite(a).all())
    z, dz = rand(g, B, S, H * D, dtype=F32), rand(g, B, S, H * D, dtype=F32)
    back = gn.rope_bwd(dz.view(B, S, H, D), f, mscale=mscale).view_as(dz)
    got = node_grads(tape_env, "Rope", [gb.tref(z, True)], [gb.tref(torch.empty_like(z))],
                     gb.rope_params(H, rot, mscale=mscale), [f.data_ptr()], dz, [(z, None)])
    assert torch.equal(got[0], back.cpu())


def test_parameter_blocks_that_end_early(gn, tape_env):
    """A block of heads, kv_heads, rot and mode alone: mscale 1, eps 1e-6."""
    gc, gb, dev = tape_env
    g = gen(9)
    x, dy = rand(g, 1, 4, 3 * 64, dtype=F32, std=1e-3), rand(g, 1, 4, 3 * 64, dtype=F32)
    f, y = freqs(64), torch.empty(1, 4, 3 * 64, device=DEV)
    full = gb.qk_norm_rope_params(1, 1, 64)
    a = node_grads(tape_env, "QkNormRope", [gb.tref(x, True)], [gb.tref(y)], full[:16], [0, 0, f.data_ptr()], dy, [(x, None)])
    b = node_grads(tape_env, "QkNormRope", [gb.tref(x, True)], [gb.tref(y)], full, [0, 0, f.data_ptr()], dy, [(x, None)])
    assert torch.equal(a[0], b[0])


def test_grouped_heads_through_the_attention(gn):
    """The documented run: fused rows of 4 + 2 + 2 heads, norms and rotation head first, k and v repeated for
    the attention, and back; fp32, against fp64 autograd within the 1e-4 of the largest element that the
    fp32 attention's own tests have (two-piece products, 2^-16 a term)."""
    g = gen(31)
    B, S, Hq, Hk, D = 2, 65, 4, 2, 64
    qkv = rand(g, B, S, (Hq + 2 * Hk) * D, dtype=F32)
    wq, wk, dO = rand(g, D, dtype=F32), rand(g, D, dtype=F32), rand(g, B, Hq, S, D, dtype=F32)
    pos = torch.randint(0, 900, (B, S), device=DEV, generator=g).to(torch.int32)
    f, m = gn.rope_freqs(D, theta=1e6, scaling="yarn", factor=4.0, trained=8192)
    q, k, v = (t.view(B, S, -1, D) for t in qkv.split((Hq * D, Hk * D, Hk * D), dim=-1))
    n = Hq // Hk
    yq, yk, yv = gn.qk_norm_rope_fwd(q, k, wq, wk, f, v=v, positions=pos, mscale=m, heads_first=True)
    rk, rv = yk.repeat_interleave(n, 1), yv.repeat_interleave(n, 1)
    O, lse = gn.attn_fwd(yq, rk, rv, rope="none")
    dyq, dyk, dyv = gn.attn_bwd(yq, rk, rv, O, dO, lse, rope="none")
    dyk, dyv = (t.view(B, Hk, n, S, D).float().sum(2).to(t.dtype) for t in (dyk, dyv))
    dq, dk, dv, dwq, dwk = gn.qk_norm_rope_bwd(dyq, dyk, q, k, wq, wk, f, dyv=dyv, positions=pos, mscale=m,
                                               heads_first=True)
    x = qkv.cpu().double().requires_grad_()
    w = [t.cpu().double().requires_grad_() for t in (wq, wk)]
    a = x.view(B, S, -1, D)
    a, b, c = a[:, :, :Hq], a[:, :, Hq:Hq + Hk], a[:, :, Hq + Hk:]
    ang = pos.cpu().double()[:, :, None, None] * f.cpu()
    cos, sin = m * torch.cos(ang), m * torch.sin(ang)

    def norm_turn(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        u, y = t.chunk(2, -1)
        return torch.cat((u * cos - y * sin, y * cos + u * sin), -1).transpose(1, 2)

    a, b, c = norm_turn(a, w[0]), norm_turn(b, w[1]).repeat_interleave(n, 1), c.transpose(1, 2).repeat_interleave(n, 1)
    s = (a @ b.transpose(-1, -2).contiguous()) * D ** -0.5
    s = s.masked_fill(torch.triu(torch.ones(S, S, dtype=torch.bool), 1), float("-inf"))
    o = torch.softmax(s, -1) @ c
    (o * dO.cpu().double()).sum().backward()
    got = torch.cat([t.reshape(B, S, -1) for t in (dq, dk, dv)], -1)
    for have, want in ((O, o.detach()), (got, x.grad), (dwq, w[0].grad), (dwk, w[1].grad)):
        assert float((have.cpu().double() - want).abs().max() / want.abs().max()) < 1e-4


def test_sizes_past_31_bits_are_refused(gn):
    x = torch.zeros(1, 1, 1, 2, device=DEV).expand(2 ** 32 + 2, 1, 1, 2)
    with pytest.raises(gn.GnError, match="31 bits"):
        gn.rope_fwd(x, freqs(2))
    with pytest.raises(gn.GnError, match="31 bits"):
        gn.qk_norm_rope_fwd(x, None)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_loss_below_a_mean(gn, tape_env, dtype):
    """LinearCrossEntropy with scale 1 and a Mean of its rows gives the gradients of the root with scale 1 / T
    (1 / T is a power of two: the same bits); another scale multiplies what comes from behind."""
    gc, gb, dev = tape_env
    g = gen(12)
    T, d, V = 64, 32, 90
    h, E = rand(g, T, d, dtype=dtype), rand(g, V, d, dtype=dtype, std=0.3)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    mean, one = loss.mean().reshape(1), torch.ones(1, device=DEV)
    for scale in (1.0, 0.5):
        dh, dE = gn.linear_xent_bwd(h, E, t, lse, scale=scale / T)
        tape = gb.create_tape_context(dev)
        tape.begin()
        n = tape.record_op(gc.OpType.LinearCrossEntropy, [gb.tref(h, True), gb.tref(t)], [gb.tref(loss)],
                           gb.linear_cross_entropy_params(V, scale))
        tape.save_for_backward(n, [E.data_ptr(), lse.data_ptr()])
        n = tape.record_op(gc.OpType.Mean, [gb.tref(loss, True)], [gb.tref(mean)])
        tape.backward(n, one.data_ptr())
        for x, dt, want in ((h, gb.dtype_code(h), dh), (E, gb.DTYPE_F32, dE)):
            got = torch.from_numpy(gb.download(dev, tape.get_grad_buffer(x.data_ptr()), x.shape, dt))
            assert torch.equal(got, want.float().cpu())
        tape.end()


@pytest.mark.parametrize("T,d", [(16, 256), (20, 512), (32, 2048), (16, 77), (64, 64), (64, 1024), (300, 72), (300, 33),
                                 (2001, 264), (4096, 264)])
def test_three_pieces_of_few_rows(gn, T, d):
    """Up to 4096 rows an fp32 dE is as good as fp32's own: equal logits, p = 1 / 512, five rows with a weight,
    three of them with one target.  lse = 9 ln 2 is off by half its step, 2^-22, and ln 2's rounding, p by
    that, exp2's 2^-23 twice and a product's 2^-24: 2^-20.  Two pieces of G, 2^-17 of an element, do not pass."""
    g = gen(T + d)
    V = 512
    h, E = rand(g, T, d), torch.zeros(V, d, device=DEV, dtype=BF)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    at = torch.tensor([1, 4, T // 2, T - 3, T - 1], device=DEV)
    t[at] = torch.tensor([7, 100, 7, 7, V - 1], device=DEV, dtype=torch.int32)
    u = torch.zeros(T, device=DEV)
    u[at] = torch.rand(5, device=DEV, generator=g) + 0.1
    lse = gn.linear_xent_fwd(h, E, t)[1]
    _, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u)
    one = torch.ones(V, d, device=DEV)
    gn.linear_xent_bwd(h, E, t, lse, dloss=u, need_dh=False, dE=one, accumulate=True)
    p = (u[at].double() / V)[:, None].expand(5, V)
    G = p.clone()
    G[torch.arange(5), t[at].long()] -= u[at].double()
    x = h[at].double()
    ref = G.t() @ x
    bound = (p * 2.0 ** -20 + G.abs() * 2.0 ** -23).t() @ x.abs() + 8 * 2.0 ** -24 * (G.t().abs() @ x.abs()) + 1e-30
    assert bool(((dE.double() - ref).abs() <= bound).all())
    assert bool(((one.double() - 1 - ref).abs() <= bound + 2 * 2.0 ** -24 * (1 + ref.abs() + bound)).all())
    first = G.float().bfloat16().double()
    two = first + (G - first).float().bfloat16().double()
    assert bool(((two.t() @ x - ref).abs() > bound).any())


@pytest.mark.parametrize("T,d", [(1, 256), (16, 256), (20, 512), (32, 2048), (16, 77), (64, 64), (128, 1024), (300, 72),
                                 (300, 33), (512, 264)])
def test_bf16_dE_of_few_rows_is_rounded_once(gn, T, d):
    """Up to 512 rows a bf16 dE takes two pieces of G: its own rounding (2^-8 of the value), and besides it
    2^-16 of G, p's 2^-20 and fp32 sums.  Equal logits, five rows with a weight.  One piece does not pass."""
    g = gen(T + d)
    V = 512
    h, E = rand(g, T, d), torch.zeros(V, d, device=DEV, dtype=BF)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    at = torch.tensor(sorted({0, T // 3, T // 2, (3 * T) // 4, T - 1}), device=DEV)
    u = torch.zeros(T, device=DEV)
    u[at] = torch.rand(len(at), device=DEV, generator=g) + 0.1
    lse = gn.linear_xent_fwd(h, E, t)[1]
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u, dE_dtype=BF)
    assert torch.equal(dh, gn.linear_xent_bwd(h, E, t, lse, dloss=u, need_dE=False)[0])
    p = (u[at].double() / V)[:, None].expand(len(at), V)
    G = p.clone()
    G[torch.arange(len(at)), t[at].long()] -= u[at].double()
    x = h[at].double()
    ref = G.t() @ x
    bound = (p * 2.0 ** -20 + G.abs() * 2.0 ** -16).t() @ x.abs() * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + 1e-30
    assert bool(((dE.double() - ref).abs() <= bound).all())
    one = (G.float().bfloat16().double().t() @ x).float().bfloat16().double()
    assert bool(((one - ref).abs() > bound).any())
