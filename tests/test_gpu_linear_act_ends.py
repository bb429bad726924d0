"""GPU tests of linear_act_fwd and act_linear_bwd where the numbers end: slopes of the largest P, NaN in a sum, fp32 activations to a
few units in the last place, and the fp32 and odd-sized backward against the plain linear layer's.

u = 2^-24.  The math library's exponential is good to one step (2 u of itself), its tanh to two (4 u), erfc to four (8 u);
a sum, product or quotient to u."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_linear_act import ACTS, BF, DEV, F32, act64, check_bwd, near, rand, slope64  # noqa: E402

U = 2.0 ** -24


@pytest.fixture(scope="module")
def gn(gpu):
    import gn_bwd
    gn_bwd.lib()
    return gn_bwd


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K", [(16, 16), (2048, 256)])
def test_slopes_of_the_largest(gn, M, K, dtype):
    """gelu's slope is 0 or 1 far out, where its argument's square and cube overflow (W is the unit matrix, dY 1)."""
    x = torch.tensor([25., 1e13, 3e18, 3e19, 3.8e36, 4e36, 1e37, 3e38], device=DEV)
    P = torch.cat((x, -x)).to(dtype).repeat(M, K // 16)
    I, dY = torch.eye(K, device=DEV, dtype=dtype), torch.ones(M, K, device=DEV, dtype=dtype)
    want = (P > 0).double()
    acts = ("relu", "gelu_tanh", "gelu_erf", "silu")
    for act in acts:
        near(gn.act_linear_bwd(act, dY, P, None, I, need_dw=False)[0], want, 2 ** -20)
    P[:, 0] = math.inf
    P[:, 8] = -math.inf
    near(gn.act_linear_bwd("gelu_tanh", dY, P, None, I, need_dw=False)[0], want, 2 ** -20)
    P[:, 3] = math.nan
    for act in acts[1:] + ("tanh", "sigmoid"):
        assert bool(torch.isnan(gn.act_linear_bwd(act, dY, P, None, I, need_dw=False)[0][:, 3]).all()), act


@pytest.mark.parametrize("act", ["none"] + ACTS)
@pytest.mark.parametrize("dtype,res", [(BF, None), (BF, F32), (F32, None), (F32, F32)])
def test_nan_in_a_sum_stays(gn, act, dtype, res):
    """A NaN among a row's inputs is in all of its outputs and in no other row's."""
    for M, N, K in ((5, 24, 16), (70, 200, 136), (700, 1024, 256), (33, 35, 37)):
        X, W, b = rand(1, M, K, dtype=dtype), rand(2, N, K, dtype=dtype, std=K ** -0.5), rand(3, N, dtype=dtype)
        R = None if res is None else rand(4, M, N, dtype=res)
        for pre in (False, True):
            clean = gn.linear_act_fwd(X, W, b, act=act, residual=R, need_pre=pre)
            Xn = X.clone()
            Xn[3, 7] = math.nan
            got = gn.linear_act_fwd(Xn, W, b, act=act, residual=R, need_pre=pre)
            for c, g in zip(clean, got) if pre else ((clean, got),):
                assert bool(torch.isnan(g[3]).all()), (M, pre)
                rest = torch.arange(M, device=DEV) != 3
                assert torch.equal(g[rest], c[rest])


def z2(x):
    """gelu_tanh's 2 z and its derivative."""
    k = 2 * math.sqrt(2 / math.pi)
    return k * (x + 0.044715 * x ** 3), k * (1 + 3 * 0.044715 * x * x)


@pytest.mark.parametrize("M,N,K", [(40, 64, 48), (500, 256, 256)])
@pytest.mark.parametrize("act", ACTS)
def test_fp32_activations(gn, act, M, N, K):
    """At the very sums (the same call without an activation).  silu, sigmoid: e^-x 2 u, 1 + it, the quotient.  tanh: the
    library's.  gelu_tanh: 2 z, of a square, two constants, a sum and a product, to 4 u of itself, which e^-2z hands on.  gelu_erf:
    erfc's argument to 2 u, and erfc hands on at most x^2 times that."""
    X, W, b = rand(1, M, K, dtype=F32), rand(2, N, K, dtype=F32, std=K ** -0.5), rand(3, N, dtype=F32)
    v = gn.linear_act_fwd(X, W, b).double()
    Y = gn.linear_act_fwd(X, W, b, act=act)
    # (1 + tanh and 1 + erf of fp64 cancel where v is far below 0)
    ref = v * torch.special.erfc(-v / math.sqrt(2)) / 2 if act == "gelu_erf" else v * torch.sigmoid(z2(v)[0]) if act == "gelu_tanh" else act64(v, act)
    size = dict(relu=0 * v, silu=4 + 0 * v, sigmoid=4 + 0 * v, tanh=4 + 0 * v, gelu_tanh=4 + 4 * z2(v)[0].abs(), gelu_erf=12 + 2 * v * v)[act]
    near(Y, ref, size * U * ref.abs())
    kept = gn.linear_act_fwd(X, W, b, act=act, need_pre=True)
    assert torch.equal(kept[0], Y) and torch.equal(kept[1], Y if act in ("tanh", "sigmoid") else v.float())


@pytest.mark.parametrize("act", ACTS)
def test_fp32_slopes(gn, act):
    """At P (W is the unit matrix, dY 1).  s + x s (1 - s) z' with s as above: its two terms' magnitudes to 8 + 4 |z| steps of u;
    the normal density's exponent to 2 u of x^2 / 2."""
    M, K = 300, 64
    P = rand(1, M, K, dtype=F32, std=2)
    if act in ("tanh", "sigmoid"):
        P = act64(P.double(), act).float()
    dP = gn.act_linear_bwd(act, torch.ones(M, K, device=DEV), P, None, torch.eye(K, device=DEV), need_dw=False)[0]
    x = P.double()
    if act in ("silu", "gelu_tanh"):
        z, dz = (x, torch.ones_like(x)) if act == "silu" else z2(x)
        s = torch.sigmoid(z)
        size = (8 + 4 * z.abs()) * (s + (x * s * torch.sigmoid(-z) * dz).abs())
        ref = s + x * s * torch.sigmoid(-z) * dz
    elif act == "gelu_erf":
        phi, t = torch.special.erfc(-x / math.sqrt(2)) / 2, x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        ref, size = phi + t, (12 + 2 * x * x) * phi + (8 + x * x) * t.abs()
    else:
        ref = slope64(x, act)
        size = 2 * ref
    near(dP, ref, size * U)


# few rows (one pass over W), one launch, ranges of the terms, and tiles that need neither
FP32 = [(1, 256, 784), (8, 1000, 512), (3, 10, 256), (64, 10, 256), (64, 256, 784), (128, 4096, 1024), (256, 6144, 768), (2000, 512, 256), (77, 33, 51)]


@pytest.mark.parametrize("M,N,K", FP32)
def test_fp32_backward_takes_the_linear_layers_products(gn, M, N, K):
    """With relu, whose slopes are 0 and 1: dP, dW and db are linear_bwd's, bit for bit."""
    dY, P, W = rand(1, M, N, dtype=F32, std=0.01), rand(2, M, K, dtype=F32), rand(3, N, K, dtype=F32, std=0.05)
    A = P.clamp(min=0)
    dX, dW, db = gn.linear_bwd(dY, A, W)
    got = gn.act_linear_bwd("relu", dY, P, A, W)
    assert torch.equal(got[0], dX * (P > 0)) and torch.equal(got[1], dW) and torch.equal(got[2], db)
    again = gn.act_linear_bwd("relu", dY, P, A, W)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    check_bwd(gn, M, N, K, "silu", F32, accumulate=True)
    only = gn.act_linear_bwd("relu", dY, P, None, W, need_dw=False)[0]
    ref = dY.double() @ W.double() * (P > 0)
    near(only, ref, 2 ** -23 * (N ** 0.5 + 8) * (dY.double().abs() @ W.double().abs()))


@pytest.mark.parametrize("M,N,K", FP32)
def test_fp32_backward_without_workspace(gn, M, N, K):
    """The call takes none: the same bits every time then too."""
    dY, P, W = rand(1, M, N, dtype=F32, std=0.01), rand(2, M, K, dtype=F32), rand(3, N, K, dtype=F32, std=0.05)
    A = P.clamp(min=0)
    out = []
    for _ in range(3):
        dP, dW, db = (torch.empty(*s, device=DEV) for s in ((M, K), (N, K), (N,)))
        rc = gn.lib().gn_act_linear_bwd(gn.ACT["relu"], dY.data_ptr(), P.data_ptr(), A.data_ptr(), W.data_ptr(), dP.data_ptr(),
                                        dW.data_ptr(), db.data_ptr(), M, N, K, gn.F32, 0, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        out.append((dP, dW, db))
    assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(o, out[0]))
    ref = dY.double() @ W.double() * (P > 0)
    near(out[0][0], ref, 2 ** -23 * (N ** 0.5 + 8) * (dY.double().abs() @ W.double().abs()))


@pytest.mark.parametrize("M,N,K", [(8192, 1027, 1031), (8192, 513, 519), (4100, 767, 769), (3000, 64, 100), (5000, 100, 64)])
def test_odd_weight_gradients_over_ranges_of_rows(gn, M, N, K):
    """Sizes whose laid-out weight gradient is a sum of partial planes, with their room in the workspace."""
    check_bwd(gn, M, N, K, "silu")
    check_bwd(gn, M, N, K, "gelu_tanh", accumulate=True, seed=7)
    dY, P, W = rand(1, M, N, std=0.01), rand(2, M, K), rand(3, N, K, std=0.05)
    first, second = (gn.act_linear_bwd("relu", dY, P, P, W) for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("shift", [1, 2])
@pytest.mark.parametrize("M,N,K", [(5, 64, 256), (64, 36, 100), (128, 512, 1024), (900, 264, 136)])
def test_fp32_backward_of_unaligned_views(gn, M, N, K, shift):
    check_bwd(gn, M, N, K, "gelu_tanh", F32, shift=shift)
    check_bwd(gn, M, N, K, "tanh", F32, shift=shift, accumulate=True)


@pytest.mark.parametrize("M,N,K", [(8, 1000, 512), (64, 10, 256), (128, 4096, 1024), (700, 513, 519)])
def test_fp32_two_at_once_and_replays(gn, M, N, K):
    dY, P, W = rand(1, M, N, dtype=F32, std=0.01), rand(2, M, K, dtype=F32), rand(3, N, K, dtype=F32, std=0.05)
    A = act64(P.double(), "silu").float()

    def call():
        return (gn.linear_act_fwd(P, W, act="gelu_erf"),) + gn.act_linear_bwd("silu", dY, P, A, W)

    ref = call()
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for k in range(4):
        dY.copy_(rand(20 + k, M, N, dtype=F32, std=0.01))
        P.copy_(rand(30 + k, M, K, dtype=F32))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
