"""GPU tests of the linear head's cross entropy without its logits (linear_xent), against plain fp64
torch: ragged and odd sizes, rows without a target, upstream gradients of loss and lse, both types
of the weight gradient, accumulation, far logits, streams, graph replays.

Tolerances, element by element, from the operator's own roundings:
  logits   fp32 sums of d products, exact from bf16 and 2^-22 each from fp32 (six-product split): off by
           at most el = (d 2^-24 + [fp32] 2^-22) sum |h||E|
  lse      the largest el of its row, and 2^-20 (1 + |l|) for exp, sum and log
  p        el + dlse + 2^-21 (|l| + |lse| + 1) of itself
  G        on the bf16 path one rounding to bf16 (2^-8), or two pieces (2^-16)
  dh, dE   their G's error times |E|, |h|, summed; fp32 sums of n terms n 2^-24 of the terms'
           magnitudes (fp32: 2^-22 each besides); the output's rounding."""
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


def guarded(g, *shape, std=1.0, dtype=BF, offset=0):
    """A tensor at element `offset` of a buffer whose other elements are NaN."""
    n = 1
    for s in shape:
        n *= s
    buf = torch.full((offset + n + 4096,), float("nan"), device=DEV, dtype=dtype)
    buf[offset:offset + n] = (torch.randn(n, device=DEV, generator=g) * std).to(dtype)
    return buf[offset:offset + n].view(*shape)


def targets(g, T, V):
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    if T > 2:
        t[1::5] = -100
        t[2] = V  # out of range is no target either
        t[0] = V - 1
    return t


class Ref:
    """Values and error bounds in fp64."""

    def __init__(self, h, E, t, u=None, z=None):
        f32 = h.dtype == F32
        (T, d), V = h.shape, E.shape[0]
        hd, Ed = h.double(), E.double()
        each = 2.0 ** -22 if f32 else 0.0
        l = hd @ Ed.t()
        el = (hd.abs() @ Ed.abs().t()) * (d * 2.0 ** -24 + each)
        self.lse = torch.logsumexp(l, -1)
        self.dlse = el.amax(-1) + 2.0 ** -20 * (1 + l.abs().amax(-1))
        ok = (t >= 0) & (t < V)
        at = t.long().clamp(0, V - 1)
        rows = torch.arange(T, device=DEV)
        self.loss = torch.where(ok, self.lse - l[rows, at], 0.0)
        self.dloss = torch.where(ok, self.dlse + el[rows, at] + 2.0 ** -23 * self.lse.abs(), 0.0)
        if u is None and z is None:
            return
        u = torch.where(ok, torch.ones(T, device=DEV, dtype=F64) if u is None else u.double(), 0.0)
        z = torch.zeros(T, device=DEV, dtype=F64) if z is None else z.double()
        p = torch.exp(l - self.lse[:, None])
        dp = p * (el + self.dlse[:, None] + 2.0 ** -21 * (l.abs() + self.lse.abs()[:, None] + 1))
        a = (u + z)[:, None]
        G = a * p
        G[rows, at] -= u
        dG = a.abs() * dp + 2.0 ** -22 * (G.abs() + a.abs() * p)

        def out(G, dG, X, n, split, eps):
            g = dG + (0 if f32 else (2.0 ** -16 if split else 2.0 ** -8) * (G.abs() + dG))
            v = G @ X
            return v, g @ X.abs() + (n * 2.0 ** -24 + each) * (G.abs() @ X.abs()) + eps * v.abs() + 1e-30

        self.dh = out(G, dG, Ed, V, False, 2.0 ** -24 if f32 else 2.0 ** -8)
        self.dE = out(G.t(), dG.t(), hd, T, True, 2.0 ** -23)
        self.dEb = out(G.t(), dG.t(), hd, T, False, 2.0 ** -8)


def within(got, ref, bound):
    assert bool(torch.isfinite(got).all())
    d = (got.double() - ref).abs()
    bad = d > bound
    assert not bool(bad.any()), (float((d / bound).max()), int(bad.sum()))


SIZES = [  # T, d, V
    (1, 8, 1), (1, 64, 50), (3, 72, 7), (2, 128, 64), (16, 64, 1000), (63, 72, 257), (65, 136, 4097), (129, 768, 2000),
    (200, 64, 33001), (257, 256, 1024), (5, 77, 131), (40, 33, 1000), (1, 770, 515), (300, 1000, 777),
    # dh of few rows over ranges of the vocabulary
    (1, 1024, 4097), (5, 520, 6200), (32, 2048, 1601), (64, 512, 6145), (97, 1024, 3401), (128, 264, 11917),
    # few rows, every width that is read in whole rows
    (1, 256, 3), (32, 512, 1003), (31, 768, 4096), (7, 1024, 129), (32, 1280, 8200), (2, 1536, 64), (17, 1792, 500),
    (16, 2048, 33000), (5, 2304, 300), (33, 256, 9000),
    # several pieces of the vocabulary, the last of any width
    (8193, 16, 33001), (8193, 12, 9001), (8193, 16, 16387), (40001, 8, 4098)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d,V", SIZES)
def test_linear_xent(gn, T, d, V, dtype):
    g = gen(T + d + V)
    h = guarded(g, T, d, dtype=dtype)
    E = guarded(g, V, d, dtype=dtype, std=3 * d ** -0.5)
    t = targets(g, T, V)
    u = torch.rand(T, device=DEV, generator=g) - 0.25
    z = torch.rand(T, device=DEV, generator=g) - 0.5
    r = Ref(h, E, t, u * 0.5, z * 0.5)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    within(lse, r.lse, r.dlse)
    within(loss, r.loss, r.dloss + 1e-30)
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u, dlse=z, scale=0.5)
    within(dh, *r.dh)
    within(dE, *r.dE)
    # one of the two alone, the same bits; onto a gradient that is there
    assert torch.equal(gn.linear_xent_bwd(h, E, t, lse, dloss=u, dlse=z, scale=0.5, need_dE=False)[0], dh)
    one = torch.ones(V, d, device=DEV)
    gn.linear_xent_bwd(h, E, t, lse, dloss=u, dlse=z, scale=0.5, need_dh=False, dE=one, accumulate=True)
    within(one, r.dE[0] + 1, r.dE[1] + 2.0 ** -23 * (1 + r.dE[0].abs()))
    if dtype == BF:
        dEb = gn.linear_xent_bwd(h, E, t, lse, dloss=u, dlse=z, scale=0.5, need_dh=False, dE_dtype=BF)[1]
        within(dEb, *r.dEb)
    # the plain loss: upstream 1
    r = Ref(h, E, t, torch.ones(T, device=DEV))
    dh, dE = gn.linear_xent_bwd(h, E, t, lse)
    within(dh, *r.dh)
    within(dE, *r.dE)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [33, 4200])
@pytest.mark.parametrize("offset", [1, 2])
def test_unaligned(gn, offset, T, dtype):
    g = gen(offset)
    h, E = guarded(g, T, 64, dtype=dtype, offset=offset), guarded(g, 300, 64, dtype=dtype, offset=offset, std=0.3)
    t = targets(g, T, 300)
    u = torch.ones(T, device=DEV)
    r = Ref(h, E, t, u)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    within(lse, r.lse, r.dlse)
    within(loss, r.loss, r.dloss + 1e-30)
    buf = torch.full((offset + 300 * 64 + 64,), 5.0, device=DEV)
    dE = buf[offset:offset + 300 * 64].view(300, 64)
    dh, _ = gn.linear_xent_bwd(h, E, t, lse, dE=dE)
    within(dh, *r.dh)
    within(dE, *r.dE)
    assert bool((buf[:offset] == 5).all()) and bool((buf[offset + 300 * 64:] == 5).all())


def test_far_logits(gn):
    """Logits of some hundreds: the running maximum keeps exp in range; a certain row has no gradient."""
    g = gen(9)
    T, d, V = 70, 64, 900
    h, E = guarded(g, T, d, std=20.0), guarded(g, V, d, std=2.0)
    t = (h.double() @ E.double().t()).argmax(-1).to(torch.int32)
    u = torch.ones(T, device=DEV)
    r = Ref(h, E, t, u)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    within(lse, r.lse, r.dlse)
    within(loss, r.loss, r.dloss + 1e-30)
    assert float(lse.max()) > 300
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u)
    within(dh, *r.dh)
    within(dE, *r.dE)


@pytest.mark.parametrize("T,d", [(4097, 64), (5001, 77), (16384, 264)])
def test_target_elements_of_many_rows(gn, T, d):
    """An fp32 dE of many rows, five of them with a weight and three of those with one target: G's target
    elements are taken whole (2^-24, not the 2^-16 of two bf16 pieces; equal logits, p = 1 / V)."""
    g = gen(T)
    V = 520
    h = guarded(g, T, d)
    E = torch.zeros(V, d, device=DEV, dtype=BF)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    at = torch.tensor([3, 700, 1500, T - 300, T - 1], device=DEV)
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
    # p: its own rounding and lse's (2^-20 (1 + lse) and 2^-21 (lse + 1)), and two pieces where it is no target
    dG = p * (2.0 ** -16 + 2.0 ** -19 * 8) + 2.0 ** -23 * G.abs()
    ref = G.t() @ x
    bound = dG.t() @ x.abs() + 8 * 2.0 ** -24 * (G.t().abs() @ x.abs()) + 1e-30
    within(dE, ref, bound)
    within(one, ref + 1, bound + 2 * 2.0 ** -24 * (1 + ref.abs() + bound))


def test_two_calls_at_once(gn):
    """Two streams, a workspace each: the bits of one call after the other."""
    g = gen(17)
    sets = []
    for T, d, V in ((4200, 256, 9001), (3000, 256, 12001)):
        h, E, t = guarded(g, T, d), guarded(g, V, d, std=0.2), targets(g, T, V)
        loss, lse = gn.linear_xent_fwd(h, E, t)
        sets.append((h, E, t, lse, gn.linear_xent_bwd(h, E, t, lse),
                     gn.workspace(gn.linear_xent_workspace_bytes(T, d, V, gn.BF16), DEV)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, (h, E, t, lse, _, ws) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(gn.linear_xent_bwd(h, E, t, lse, ws=ws))
    torch.cuda.synchronize()
    for i in range(2):
        for dh, dE in got[i]:
            assert torch.equal(dh, sets[i][4][0]) and torch.equal(dE, sets[i][4][1])


def test_no_row_has_a_target(gn):
    g = gen(10)
    h, E = guarded(g, 20, 64), guarded(g, 100, 64)
    t = torch.full((20,), -100, device=DEV, dtype=torch.int32)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    assert bool((loss == 0).all()) and bool(torch.isfinite(lse).all())
    dh, dE = gn.linear_xent_bwd(h, E, t, lse)
    assert bool((dh == 0).all()) and bool((dE == 0).all())


def test_one_bad_row_stays_alone(gn):
    """A row of h with NaN or inf spoils its own loss and dh only."""
    g = gen(12)
    h, E = guarded(g, 40, 64), guarded(g, 300, 64)
    t = targets(g, 40, 300)
    good, glse = gn.linear_xent_fwd(h, E, t)
    gdh, _ = gn.linear_xent_bwd(h, E, t, glse, need_dE=False)
    h[7] = float("nan")
    loss, lse = gn.linear_xent_fwd(h, E, t)
    dh, _ = gn.linear_xent_bwd(h, E, t, lse, need_dE=False)
    rest = [i for i in range(40) if i != 7]
    assert bool(torch.isnan(lse[7])) and torch.equal(loss[rest], good[rest]) and torch.equal(lse[rest], glse[rest])
    assert torch.equal(dh[rest], gdh[rest]) and bool(torch.isnan(dh[7]).all())


def test_empty(gn):
    E = guarded(gen(1), 30, 64)
    h = torch.empty(0, 64, device=DEV, dtype=BF)
    t = torch.empty(0, device=DEV, dtype=torch.int32)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    assert loss.shape == lse.shape == (0,)
    dh, dE = gn.linear_xent_bwd(h, E, t, lse)
    assert dh.shape == (0, 64) and bool((dE == 0).all())
    one = torch.ones(30, 64, device=DEV)
    gn.linear_xent_bwd(h, E, t, lse, dE=one, accumulate=True)
    assert bool((one == 1).all())


def test_gradient_against_differences(gn):
    """fp32: the slope of sum(u loss + z lse) along a random direction of h and E."""
    g = gen(14)
    T, d, V = 12, 24, 90
    h, E = guarded(g, T, d, dtype=F32), guarded(g, V, d, dtype=F32, std=0.5)
    t = targets(g, T, V)
    u, z = torch.rand(T, device=DEV, generator=g), torch.rand(T, device=DEV, generator=g)

    def value(h, E):
        loss, lse = gn.linear_xent_fwd(h, E, t)
        return float((u.double() * loss + z.double() * lse).sum())

    dh, dE = gn.linear_xent_bwd(h, E, t, gn.linear_xent_fwd(h, E, t)[1], dloss=u, dlse=z)
    a, b = torch.randn(T, d, device=DEV, generator=g), torch.randn(V, d, device=DEV, generator=g)
    s = 2.0 ** -8
    slope = (value(h + s * a, E + s * b) - value(h - s * a, E - s * b)) / (2 * s)
    want = float((dh.double() * a).sum() + (dE.double() * b).sum())
    # 24 values of up to 20, each good to 2^-19, over the step; the third difference
    assert abs(slope - want) <= 24 * 20 * 2.0 ** -19 / s + 1e-2 * abs(want)


def test_against_the_framework_s_own_path(gn):
    """Linear, xent_bwd over stored logits and linear_bwd give the same gradients (fp32)."""
    g = gen(15)
    T, d, V = 50, 64, 500
    h, E = guarded(g, T, d, dtype=F32).contiguous(), guarded(g, V, d, dtype=F32, std=0.3).contiguous()
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    dl = gn.xent_bwd(gn.linear_fwd(h, E), t, scale=1.0 / T)
    dh0, dE0, _ = gn.linear_bwd(dl, h, E, need_db=False)
    _, lse = gn.linear_xent_fwd(h, E, t)
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, scale=1.0 / T)
    assert float((dh - dh0).abs().max() / dh0.abs().max()) < 1e-5
    assert float((dE - dE0).abs().max() / dE0.abs().max()) < 1e-5


@pytest.mark.parametrize("T,d,V", [(130, 128, 3001), (12, 512, 7000), (60, 1024, 4001), (4200, 128, 3001), (4200, 33, 700)])
def test_on_another_stream_and_replayed(gn, T, d, V):
    g = gen(16)
    h, E = guarded(g, T, d).contiguous(), guarded(g, V, d, std=0.2).contiguous()
    t = targets(g, T, V)
    u = torch.rand(T, device=DEV, generator=g)

    def both(ws):
        loss, lse = gn.linear_xent_fwd(h, E, t, ws=ws)
        return (loss, lse, *gn.linear_xent_bwd(h, E, t, lse, dloss=u, ws=ws))

    nb = gn.linear_xent_workspace_bytes(T, d, V, gn.BF16)
    ws = gn.workspace(nb, DEV)
    eager = both(ws)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = both(gn.workspace(nb, DEV))
    s.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(ws)
    for i in range(3):
        h.copy_(torch.randn(T, d, device=DEV, generator=gen(40 + i)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(both(None), held):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [16, 40])
def test_offsets_past_32_bits(gn, T):
    """A vocabulary whose E and dE have more than 2^31 elements, some rows' targets behind them."""
    g = gen(T)
    d, V = 2048, 1100001
    h = guarded(g, T, d)
    E = torch.empty(V, d, device=DEV, dtype=BF)
    for v in range(0, V, 100000):
        E[v:v + 100000].normal_(0, 0.02, generator=g)
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    t[:4] = torch.tensor([V - 1, 1048576, 1048577, 0], dtype=torch.int32)
    hd = h.double()
    l = torch.cat([hd @ E[v:v + 100000].double().t() for v in range(0, V, 100000)], 1)
    el = d * 2.0 ** -24 * (hd.abs() @ E.float().abs().amax(0).double()[:, None])  # at least sum |h||E| of each logit
    lse = torch.logsumexp(l, -1)
    dlse = el[:, 0] + 2.0 ** -20 * (1 + l.abs().amax(-1))
    rows = torch.arange(T, device=DEV)
    loss, got = gn.linear_xent_fwd(h, E, t)
    within(got, lse, dlse)
    within(loss, lse - l[rows, t.long()], dlse + el[:, 0] + 2.0 ** -23 * lse.abs())
    dh, dE = gn.linear_xent_bwd(h, E, t, got, scale=0.5)
    p = 0.5 * torch.exp(l - lse[:, None])
    dp = p * (el + dlse[:, None] + 2.0 ** -21 * (l.abs() + lse.abs()[:, None] + 1))
    G = p
    G[rows, t.long()] -= 0.5
    dG = dp + 2.0 ** -22 * (G.abs() + 0.5)
    ref, bound = torch.zeros(T, d, device=DEV, dtype=F64), torch.zeros(T, d, device=DEV, dtype=F64)
    for v in range(0, V, 100000):
        at = slice(v, v + 100000)
        Ed = E[at].double()
        ref += G[:, at] @ Ed
        # G in bf16, the fp32 sum of V terms in ranges of a few thousand
        bound += (dG[:, at] + (2.0 ** -8 + 2.0 ** -11) * G[:, at].abs()) @ Ed.abs()
    within(dh, ref, bound + 2.0 ** -8 * ref.abs())
    for at in (slice(0, 300), slice(1048500, 1048700), slice(V - 300, V)):
        X = G[:, at].t()
        within(dE[at], X @ hd, (dG[:, at].t() + (2.0 ** -16 + T * 2.0 ** -24) * X.abs()) @ hd.abs() + 1e-30)
    assert bool(torch.isfinite(dE[::1000]).all())
