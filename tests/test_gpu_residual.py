"""GPU tests of dropout and of the residual branch (residual_norm: norms, gate, dropout, residual sum), against
plain torch in fp64: types, widths, gates, masks that drop everything, in-place use, accumulation,
streams, graph replays.

Tolerances, element by element.  Rounding to the output type: half a step, finfo.eps / 2 of the value.
Before it, in fp32 (half a step: 2^-24): a row's sum of F <= 9001 terms has at most 18 roundings in a lane's chain
where a lane holds the row (24 in the wide kernel) and 6 + 16 behind it, so a mean is within 2^-18 of the mean of
magnitudes and r within 2^-18 of itself, with its reciprocal root; a norm adds four roundings, so what it gives is
within 2^-17 (|v^| + r mean|v|) |w| + 2^-23 |b|.  A norm of a value that carries an error of itself passes
that on times r |w| (1 + |v^| + 1).  A gradient's terms d, mean and v^ mean are each good to 2^-16 of
their magnitudes' sum; every stage behind doubles that at most.  Sums over rows add their terms' errors and
at most 2^-24 (rows) of the terms' magnitudes."""
import numpy as np
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


def rand(seed, *shape, dtype=BF, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def factors(p, n, seed, stream, step, first=0):
    """fp64 factors of elements first, first + 1, ...: numpy's unsigned integers, as the header has them."""
    u64 = np.uint64

    def mix(z):
        z = (z ^ (z >> u64(30))) * u64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> u64(27))) * u64(0x94D049BB133111EB)
        return z ^ (z >> u64(31))

    phi, one = u64(0x9E3779B97F4A7C15), np.ones(1, u64)
    with np.errstate(over="ignore"):
        key = mix(mix(one * u64(seed) + phi * (one * u64(stream) + u64(1))) + phi * (one * u64(step) + u64(1)))
        i = np.arange(first, first + n, dtype=u64)
        w = mix(key + phi * ((i >> u64(1)) + u64(1)))
    half = np.where(i & u64(1), w >> u64(32), w & u64(0xffffffff))
    t = round(p * 2 ** 32)
    return torch.from_numpy((half >= u64(t)) / (1 - t / 2 ** 32)).to(DEV)


def near(got, ref, size):
    """|got - ref| <= its type's rounding of ref + size."""
    e = torch.finfo(got.dtype).eps / 2
    d = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    bad = d > e * ref.abs() + size + torch.finfo(got.dtype).tiny
    assert not bool(bad.any()), (float((d / (e * ref.abs() + size + 1e-300)).max()), int(bad.sum()))


# ---- dropout -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 511, 4096, 4099, 100003])
def test_dropout(gn, n, dtype):
    x = rand(n, n, dtype=dtype)
    for p, seed, stream, step in ((0.1, 5, 0, 0), (0.5, 2 ** 64 - 1, 3, 2 ** 63 + 5), (0.999, 1, 2 ** 40, 7), (0.0, 9, 9, 9)):
        ref = x.double() * factors(p, n, seed, stream, step)
        kept = ref != 0
        got = gn.dropout_fwd(x, p, seed, stream, step)
        near(got, ref, 2 ** -23 * ref.abs())  # the factor and the product: two half steps
        assert bool((got[~kept] == 0).all())
        assert torch.equal(gn.dropout_bwd(x, p, seed, stream, step), got)
        at = torch.tensor([step - 2 ** 64 if step >= 2 ** 63 else step], device=DEV)
        assert torch.equal(gn.dropout_fwd(x, p, seed, stream, at), got)
        same = x.clone()
        assert gn.dropout_fwd(same, p, seed, stream, step, out=same) is same and torch.equal(same, got)
        into = rand(n + 1, n, dtype=dtype)
        was = into.double()
        gn.dropout_bwd(x, p, seed, stream, step, out=into, accumulate=True)
        near(into, ref + was, 2 ** -22 * (ref.abs() + was.abs()))


def test_dropout_unaligned_and_zero_size(gn):
    x = rand(3, 1003)
    for off in (1, 3, 4):
        got = gn.dropout_fwd(x[off:], 0.3, 11)
        assert torch.equal(got, gn.dropout_fwd(x[off:].clone(), 0.3, 11))
    assert gn.dropout_fwd(x[:0], 0.3, 11).numel() == 0


def test_dropped_inf_and_nan_are_zero(gn):
    for v in (float("inf"), float("nan"), -float("inf")):
        x = torch.full((4096,), v, device=DEV, dtype=BF)
        m = factors(0.5, 4096, 1, 2, 3) != 0
        got = gn.dropout_fwd(x, 0.5, 1, 2, 3)
        assert bool((got[~m] == 0).all()) and not bool(torch.isfinite(got[m]).any())


def test_dropout_rate_and_independence(gn):
    """The share kept, and that masks of neighbouring seeds, streams and steps agree as often as independent
    ones: within 6 standard deviations of 2^20 draws."""
    n = 1 << 20
    x = torch.ones(n, device=DEV)
    for p in (0.1, 0.5):
        base = gn.dropout_fwd(x, p, 7, 1, 1) != 0
        sd = (p * (1 - p) / n) ** 0.5
        assert abs(float(base.double().mean()) - (1 - p)) < 6 * sd
        same = p * p + (1 - p) ** 2
        for other in ((8, 1, 1), (7, 2, 1), (7, 1, 2), (7, 0, 2)):
            m = gn.dropout_fwd(x, p, *other) != 0
            assert abs(float((m == base).double().mean()) - same) < 6 * (same * (1 - same) / n) ** 0.5
        assert abs(float((base[1:] == base[:-1]).double().mean()) - same) < 6 * (same * (1 - same) / n) ** 0.5


def test_dropout_past_32_bits(gn):
    n = (1 << 32) + 24
    x = torch.ones(n, device=DEV, dtype=BF)
    gn.dropout_fwd(x, 0.5, 3, 4, 5, out=x)
    for first in (0, (1 << 31) - 8, (1 << 32) - 16, n - 32):
        assert torch.equal(x[first:first + 32].double(), factors(0.5, 32, 3, 4, 5, first))


def test_dropout_replays_read_the_step(gn):
    x = rand(1, 5000)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    y = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gn.dropout_fwd(x, 0.4, 6, 1, step, out=y)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gn.dropout_fwd(x, 0.4, 6, 1, step, out=y)
    for k in range(4):
        step.fill_(k)
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, gn.dropout_fwd(x, 0.4, 6, 1, k))
        torch.cuda.synchronize()


# ---- the residual branch ---------------------------------------------------------------------
def stats(v, kind, eps):
    """v^, r and the mean magnitude of a row."""
    if kind == "none":
        return v, torch.ones_like(v[:, :1]), torch.zeros_like(v[:, :1])
    size = v.abs().mean(-1, keepdim=True)
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    else:
        size = torch.zeros_like(size)
    r = ((v * v).mean(-1, keepdim=True) + eps).rsqrt()
    return v * r, r, r * size


EPS = {"none": 0.0, "rms": 1e-6, "layer": 1e-5}


class Case:
    def __init__(self, rows, F, post="none", pre="layer", gates=0, p=0.0, x=F32, h=BF, bias=True, weights=True, seed=0,
                 scale=0.7, res_scale=0.9):
        self.rows, self.F, self.post, self.pre, self.gates, self.p, self.scale, self.res_scale = \
            rows, F, post, pre, gates, p, scale, res_scale
        self.h = rand(seed, rows, F, dtype=h)
        self.x = (rand(seed + 1, rows, F, dtype=F32) * 2 + 0.5).to(x)
        w = lambda k, on: (1 + rand(seed + k, F, dtype=F32, std=0.2)).to(h) if on else None  # noqa: E731
        self.post_w, self.pre_w = w(2, post != "none" and weights), w(3, pre != "none" and weights)
        self.post_b = rand(seed + 4, F, dtype=h) if post == "layer" and bias else None
        self.pre_b = rand(seed + 5, F, dtype=h) if pre == "layer" and bias else None
        self.gate = rand(seed + 6, gates, F, dtype=h) if gates else None
        self.dy = rand(seed + 7, rows, F, dtype=x, std=0.01)
        self.dz = rand(seed + 8, rows, F, dtype=h, std=0.01) if pre != "none" else None
        self.kw = dict(post=post, post_w=self.post_w, post_b=self.post_b, pre=pre, pre_w=self.pre_w, pre_b=self.pre_b,
                       gate=self.gate, scale=scale, res_scale=res_scale, p=p, seed=77, stream=3, step=12)
        self.m = factors(p, rows * F, 77, 3, 12).view(rows, F)

    def weights(self):
        d = lambda t, v: torch.full((self.F,), v, dtype=F64, device=DEV) if t is None else t.double()  # noqa: E731
        g = torch.ones(1, self.F, dtype=F64, device=DEV) if self.gate is None else self.gate.double()
        return d(self.post_w, 1.), d(self.post_b, 0.), d(self.pre_w, 1.), d(self.pre_b, 0.), \
            g.repeat_interleave(self.rows // g.shape[0], 0)

    def check_fwd(self, y, z):
        wp, bp, wn, bn, g = self.weights()
        v, r, s = stats(self.h.double(), self.post, EPS[self.post])
        n = v * wp + bp
        en = 2 ** -17 * (v.abs() + s) * wp.abs() + 2 ** -23 * bp.abs()
        t = self.scale * g * self.m
        ref = self.res_scale * self.x.double() + t * n
        ey = 2 ** -22 * (self.res_scale * self.x.double()).abs() + t.abs() * (en + 2 ** -21 * n.abs())
        near(y, ref, ey)
        if self.pre == "none":
            assert z is None
            return
        v, r, s = stats(ref, self.pre, EPS[self.pre])
        passed = r * (ey + ey.mean(-1, keepdim=True)) + v.abs() * r * ey.amax(-1, keepdim=True)
        near(z, v * wn + bn, (2 ** -17 * (v.abs() + s) + passed) * wn.abs() + 2 ** -23 * bn.abs())

    def check_bwd(self, got, y, dy, dz, add=(0,) * 5):
        """got: residual_norm_bwd's seven at the stream y; add: what the parameters' gradients were added onto."""
        dh, dx, dgate, dpw, dpb, dnw, dnb = got
        wp, bp, wn, bn, g = self.weights()
        zero = torch.zeros(self.rows, self.F, dtype=F64, device=DEV)
        d = zero if dy is None else dy.double()
        size = d.abs()
        sums = lambda term, e, n: (term.sum(0), (e + 2 ** -24 * self.rows * term.abs()).sum(0))  # noqa: E731
        if dz is not None:
            q = dz.double()
            u, e1 = self.norm_grad(y.double(), self.pre, q * wn, 2 ** -16 * (q * wn).abs())
            d, size = d + u, size + e1 * 2 ** 16
            v, r, s = stats(y.double(), self.pre, EPS[self.pre])
            if dnw is not None:
                ref, e = sums(q * v, 2 ** -17 * (v.abs() + s) * q.abs(), 0)
                near(dnw, ref + add[3], e + 2 ** -23 * abs(add[3]))
            if dnb is not None:
                ref, e = sums(q, zero, 0)
                near(dnb, ref + add[4], e + 2 ** -23 * abs(add[4]))
        ed = 2 ** -16 * size
        if dx is not None:
            near(dx, self.res_scale * d, 2 * abs(self.res_scale) * ed)
        v, r, s = stats(self.h.double(), self.post, EPS[self.post])
        n, en = v * wp + bp, 2 ** -17 * (v.abs() + s) * wp.abs() + 2 ** -23 * bp.abs()
        t = self.scale * self.m * d
        et = 2 * abs(self.scale) * self.m * ed
        if dgate is not None:
            G = self.gates
            ref = (t * n).view(G, -1, self.F).sum(1)
            e = (2 * (et * n.abs() + t.abs() * en) + 2 ** -24 * (self.rows // G + 2) * (t * n).abs()).view(G, -1, self.F).sum(1)
            near(dgate.view(G, self.F), ref + add[0], e + 2 ** -23 * abs(add[0]))
        dn, edn = g * t, 2 * g.abs() * et
        if dpw is not None:
            ref, e = sums(dn * v, edn * v.abs() + 2 ** -16 * (v.abs() + s) * dn.abs(), 0)
            near(dpw, ref + add[1], e + 2 ** -23 * abs(add[1]))
        if dpb is not None:
            ref, e = sums(dn, edn, 0)
            near(dpb, ref + add[2], e + 2 ** -23 * abs(add[2]))
        if dh is not None:
            if self.post != "none":
                dn, edn = self.norm_grad(self.h.double(), self.post, dn * wp, 2 * edn * wp.abs())
            near(dh, dn, 2 * edn + 2 ** -22 * dn.abs())

    @staticmethod
    def norm_grad(x, kind, g, eg):
        """The gradient of a norm's input at the scaled upstream g, and its error where g's is eg."""
        v, r, s = stats(x, kind, EPS[kind])
        mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
        layer = kind == "layer"
        ref = r * (g - v * mean(g * v) - (mean(g) if layer else 0))
        ag = eg + 2 ** -17 * g.abs()
        w = v.abs() + s
        e = r * (ag + w * mean(ag * w) + 2 ** -16 * w * mean(g.abs() * w) + (mean(ag) + 2 ** -17 * mean(g.abs()) if layer else 0))
        return ref, e


KINDS = ["none", "rms", "layer"]
TYPES = [(F32, BF), (BF, BF), (F32, F32)]


@pytest.mark.parametrize("x,h", TYPES)
@pytest.mark.parametrize("post", KINDS)
@pytest.mark.parametrize("pre", KINDS)
def test_kinds(gn, post, pre, x, h):
    for rows, F, gates, p in ((5, 768, 0, 0.0), (12, 768, 3, 0.3), (9, 100, 1, 0.5), (1, 33, 1, 0.0), (40, 2048, 40, 0.1)):
        c = Case(rows, F, post, pre, gates, p, x, h)
        c.check_fwd(*gn.residual_norm_fwd(c.h, c.x, **c.kw))
        c.check_bwd(gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw), c.x, c.dy, c.dz)


@pytest.mark.parametrize("F", [1, 2, 8, 31, 64, 511, 512, 520, 1024, 1027, 1032, 2048, 2056, 4095, 4096, 4104, 8192, 8200, 9001])
@pytest.mark.parametrize("rows", [1, 7, 300])
def test_widths(gn, rows, F):
    for x, h in TYPES[:2]:
        c = Case(rows, F, "rms", "layer", 1, 0.1, x, h)
        c.check_fwd(*gn.residual_norm_fwd(c.h, c.x, **c.kw))
        c.check_bwd(gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw), c.x, c.dy, c.dz)


@pytest.mark.parametrize("F", [64, 1536, 4096, 9000])
@pytest.mark.parametrize("rows,gates", [(600, 2), (600, 7 * 3), (600, 200), (600, 300), (600, 600), (4100, 1), (4100, 2), (4100, 4100)])
def test_gates(gn, rows, gates, F):
    if rows % gates:
        rows = rows // gates * gates
    c = Case(rows, F, "layer", "rms", gates, 0.1, BF, BF)
    c.check_fwd(*gn.residual_norm_fwd(c.h, c.x, **c.kw))
    got = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
    c.check_bwd(got, c.x, c.dy, c.dz)
    again = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
    assert all(a is None if b is None else torch.equal(a, b) for a, b in zip(got, again))  # the same bits
    # without the gate's gradient the others' rows are split as without a gate
    grads = (None,) + tuple(None if t is None else torch.empty_like(t) for t in got[3:])
    c.check_bwd(gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, grads=grads, **c.kw), c.x, c.dy, c.dz)


@pytest.mark.parametrize("F", [768, 1001, 9000])
def test_parts_left_out(gn, F):
    c = Case(37, F, "layer", "layer", 1, 0.2, F32, BF, bias=False)
    call = lambda dy=c.dy, dz=c.dz, **kw: gn.residual_norm_bwd(dy, dz, c.h, c.x, **c.kw, **kw)  # noqa: E731
    full = call()
    assert full[4] is None and full[6] is None
    c.check_bwd(full, c.x, c.dy, c.dz)
    only = call(need_dh=False, need_param=False)
    assert only[0] is None and only[2:] == (None,) * 5 and torch.equal(only[1], full[1])
    only = call(need_dx=False, need_param=False)
    assert only[1] is None and torch.equal(only[0], full[0])
    c.check_bwd(call(dy=None), c.x, None, c.dz)
    got = call(dz=None)
    assert bool((got[5] == 0).all())
    c.check_bwd(got[:5] + (None, None), c.x, c.dy, None)
    bare = Case(37, F, "layer", "layer", 0, 0.0, F32, BF, bias=False, weights=False)
    bare.check_fwd(*gn.residual_norm_fwd(bare.h, bare.x, **bare.kw))
    bare.check_bwd(gn.residual_norm_bwd(bare.dy, bare.dz, bare.h, bare.x, **bare.kw), bare.x, bare.dy, bare.dz)


@pytest.mark.parametrize("rows,F,gates", [(5, 768, 1), (500, 768, 4), (500, 768, 500), (300, 1003, 2), (70, 9000, 7), (3, 9000, 0)])
def test_in_place_and_accumulate(gn, rows, F, gates):
    c = Case(rows, F, "layer", "layer", gates, 0.1, F32, BF)
    y, z = gn.residual_norm_fwd(c.h, c.x, **c.kw)
    stream = c.x.clone()
    y2, z2 = gn.residual_norm_fwd(c.h, stream, out=stream, **c.kw)
    assert y2 is stream and torch.equal(stream, y) and torch.equal(z, z2)
    ref = gn.residual_norm_bwd(c.dy, c.dz, c.h, y, **c.kw)
    onto = [None if t is None else rand(50 + i, *t.shape, dtype=F32) for i, t in enumerate(ref[2:])]
    add = [0 if t is None else t.double() for t in onto]
    dy = c.dy.clone()
    got = gn.residual_norm_bwd(dy, c.dz, c.h, y, dx=dy, grads=onto, accumulate=True, **c.kw)
    assert got[1] is dy and torch.equal(dy, ref[1]) and torch.equal(got[0], ref[0])
    c.check_bwd(got, y, c.dy, c.dz, add)


def test_unaligned_views(gn):
    """Rows of a width that vectors divide, from addresses that they do not."""
    c = Case(21, 256, "rms", "layer", 3, 0.1, BF, BF)

    def shifted(t):
        return None if t is None else torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)

    kw = {k: shifted(v) if isinstance(v, torch.Tensor) else v for k, v in c.kw.items()}
    c.check_fwd(*gn.residual_norm_fwd(shifted(c.h), shifted(c.x), **kw))
    c.check_bwd(gn.residual_norm_bwd(shifted(c.dy), shifted(c.dz), shifted(c.h), shifted(c.x), **kw), c.x, c.dy, c.dz)


def test_everything_dropped(gn):
    """A mask that leaves nothing: y is the scaled stream, the branch's gradients are 0."""
    c = Case(16, 64, "rms", "rms", 1, 1 - 2.0 ** -31, F32, BF)
    assert float(c.m.abs().max()) == 0
    y, z = gn.residual_norm_fwd(c.h, c.x, **c.kw)
    c.check_fwd(y, z)
    got = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
    assert all(float(t.abs().max()) == 0 for t in (got[0], got[2], got[3]))
    c.check_bwd(got, c.x, c.dy, c.dz)


def test_rows_do_not_touch_each_other(gn):
    """A row with inf and NaN leaves the others' results as they are; constant rows and rows of zeros give finite ones."""
    c = Case(40, 768, "layer", "layer", 0, 0.0, F32, BF)
    y, z = gn.residual_norm_fwd(c.h, c.x, **c.kw)
    g = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
    h, x = c.h.clone(), c.x.clone()
    h[3, 5], x[7] = float("nan"), float("inf")
    h[11], x[12] = 0, 0
    h[13] = 3.0
    y2, z2 = gn.residual_norm_fwd(h, x, **c.kw)
    g2 = gn.residual_norm_bwd(c.dy, c.dz, h, x, **c.kw)
    keep = [i for i in range(40) if i not in (3, 7, 11, 12, 13)]
    for a, b in ((y, y2), (z, z2), (g[0], g2[0]), (g[1], g2[1])):
        assert torch.equal(a[keep], b[keep])
        assert bool(torch.isfinite(b[[11, 12, 13]]).all())


@pytest.mark.parametrize("gates", [0, 1, 5, 40])
@pytest.mark.parametrize("F", [64, 1001, 2048, 6000, 9000])
def test_dropped_inf_and_nan_add_nothing(gn, F, gates):
    """Without a norm after the block, what the mask drops reaches no output, the gate's gradient included."""
    c = Case(40, F, "none", "layer", gates, 0.4, F32, BF)
    off = (c.m == 0).view(40, F)
    h0, h = c.h.masked_fill(off, 0.0), c.h.masked_fill(off, float("nan"))
    h[::2] = c.h.masked_fill(off, float("-inf"))[::2]
    y, z = gn.residual_norm_fwd(h0, c.x, **c.kw)
    for a, b in zip(gn.residual_norm_fwd(h, c.x, **c.kw), (y, z)):
        assert torch.equal(a, b)
    ref = gn.residual_norm_bwd(c.dy, c.dz, h0, y, **c.kw)
    for a, b in zip(gn.residual_norm_bwd(c.dy, c.dz, h, y, **c.kw), ref):
        assert a is b is None or torch.equal(a, b)
    assert (ref[2] is not None) == (gates > 0)


@pytest.mark.parametrize("rows", [1, 3, 9, 17, 33])
def test_no_eps(gn, rows):
    """Norms without an eps: lanes that have no row add nothing, not 0 / 0."""
    for F in (64, 1000, 4096, 9000):
        c = Case(rows, F, "rms", "rms", 1, 0.0, F32, BF)
        kw = dict(c.kw, post_eps=0.0, pre_eps=0.0)
        ref = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
        for a, b in zip(gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **kw), ref):
            assert a is b is None or float((a.double() - b.double()).norm()) <= 2 ** -7 * float(b.double().norm())


def test_no_rows(gn):
    c = Case(4, 64, "layer", "layer", 2)
    cut = lambda t: t[:0]  # noqa: E731
    y, z = gn.residual_norm_fwd(cut(c.h), cut(c.x), **c.kw)
    assert y.shape == z.shape == (0, 64)
    got = gn.residual_norm_bwd(cut(c.dy), cut(c.dz), cut(c.h), cut(c.x), **c.kw)
    assert all(float(t.abs().max()) == 0 for t in got[2:])


def test_elements_past_31_bits(gn):
    rows, F = (1 << 18) + 3, 8192
    h = torch.empty(rows, F, device=DEV, dtype=BF)
    x = torch.empty_like(h)
    for i in range(0, rows, 1 << 14):
        h[i:i + (1 << 14)] = rand(i, 1, F)
        x[i:i + (1 << 14)] = rand(i + 1, 1, F)
    tail = slice(rows - 5, rows)
    h[tail], x[tail] = rand(1, 5, F), rand(2, 5, F)
    w = 1 + rand(3, F, std=0.1)
    kw = dict(post="rms", post_w=w, pre="rms", pre_w=w, p=0.5, seed=1, stream=2, step=3)
    y, z = gn.residual_norm_fwd(h, x, **kw)
    m = factors(0.5, 5 * F, 1, 2, 3, (rows - 5) * F).view(5, F)
    v, r, s = stats(h[tail].double(), "rms", 1e-6)
    ref = x[tail].double() + m * v * w.double()
    near(y[tail], ref, 2 ** -16 * (x[tail].double().abs() + (m * v * w.double()).abs()))
    dh, dx, _, dpw, _, dnw, _ = gn.residual_norm_bwd(y, z, h, y, **kw)
    one = {k: v for k, v in kw.items() if k != "p"}
    last = gn.residual_norm_bwd(y[tail].contiguous(), z[tail].contiguous(), h[tail].contiguous(), y[tail].contiguous(), **one)
    assert torch.equal(dx[tail], last[1])  # the mask does not reach dx


def test_another_stream_and_replays(gn):
    c = Case(333, 1024, "rms", "layer", 1, 0.2, F32, BF)
    step = torch.tensor([12], device=DEV)
    kw = dict(c.kw, step=step)
    ref = gn.residual_norm_fwd(c.h, c.x, **c.kw)
    back = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **c.kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, z = gn.residual_norm_fwd(c.h, c.x, **kw)
        got = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **kw)
    s.synchronize()
    assert torch.equal(y, ref[0]) and torch.equal(z, ref[1])
    assert all(a is None if b is None else torch.equal(a, b) for a, b in zip(got, back))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, z = gn.residual_norm_fwd(c.h, c.x, **kw)
        got = gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **kw)
    for k in (12, 40, 12, 41):
        step.fill_(k)
        g.replay()
        torch.cuda.synchronize()
        now = dict(c.kw, step=k)
        want = gn.residual_norm_fwd(c.h, c.x, **now) + gn.residual_norm_bwd(c.dy, c.dz, c.h, c.x, **now)
        torch.cuda.synchronize()
        assert all(a is None if b is None else torch.equal(a, b) for a, b in zip((y, z) + tuple(got), want))


def test_gradients_against_differences(gn):
    """The whole backward against differences of the forward in fp32: a step e of a parameter along a direction changes
    sum(y a) + sum(z b) by e times the gradient along it, up to e^2 and the forward's roundings."""
    rows, F = 24, 96
    c = Case(rows, F, "layer", "layer", 2, 0.25, F32, F32, seed=9)
    a, b = rand(60, rows, F, dtype=F32), rand(61, rows, F, dtype=F32)
    y, _ = gn.residual_norm_fwd(c.h, c.x, **c.kw)
    grads = dict(zip(("h", "x", "gate", "post_w", "post_b", "pre_w", "pre_b"), gn.residual_norm_bwd(a, b, c.h, y, **c.kw)))
    at = dict(h=c.h, x=c.x, **{k: c.kw[k] for k in ("gate", "post_w", "post_b", "pre_w", "pre_b")})

    def value(name, e, v):
        t = dict(at)
        t[name] = t[name] + e * v
        kw = dict(c.kw, **{k: t[k] for k in ("gate", "post_w", "post_b", "pre_w", "pre_b")})
        y, z = gn.residual_norm_fwd(t["h"], t["x"], **kw)
        return float((y.double() * a.double()).sum() + (z.double() * b.double()).sum())

    for i, (name, t) in enumerate(at.items()):
        v = rand(70 + i, *t.shape, dtype=F32)
        e = 2.0 ** -6
        slope = (8 * (value(name, e, v) - value(name, -e, v)) - (value(name, 2 * e, v) - value(name, -2 * e, v))) / (12 * e)
        exact = float((grads[name].double() * v.double()).sum())
        size = float((grads[name].double() * v.double()).abs().sum())
        # the forward's roundings: 2 rows F terms of about 2^-20 each, in random order, over 12 e / 18
        noise = 18 * 2 ** -20 * (2 * rows * F) ** 0.5 * 4 / (12 * e)
        assert abs(slope - exact) < noise + 2 ** -10 * size, (name, slope, exact, size, noise)
