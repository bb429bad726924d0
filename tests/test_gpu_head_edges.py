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
