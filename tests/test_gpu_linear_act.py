"""GPU tests of linear layers with bias, activation and residual in their epilogue (linear_act_fwd) and of the
backward through the activation in front (act_linear_bwd), against plain torch in fp64: every activation and type,
few rows and many, odd sizes, unaligned views, in-place use, accumulation, streams, graph replays.

Tolerances, element by element.  Rounding to the output type: half a step, finfo.eps / 2 of the value.
Before it: a product of K terms in fp32 (bf16 operands are exact in it) is within 2^-23 (sqrt K + 8)
sum |x w| of the sum: its partial sums' roundings, half a step each and one per term at most, in random
directions, six standard deviations of which sqrt K steps are more than; the truncating adds of the matrix unit
take one step for half a one.  The fp32 products' own limit is 2^-24 a term beside that.  An activation's slope is at
most 1.13 in magnitude, so it hands on at most 1.13 times that, and adds its own: e^x to |x| 2^-23 +
2^-22 of itself, which moves what follows by at most 2^-20 (1 + |x|), tanh's and sigmoid's forms alike.  A derivative moves by
at most 0.8 per unit of its argument and errs by 2^-19 (1 + |x|) itself."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"
ACTS = ["relu", "gelu_tanh", "gelu_erf", "silu", "tanh", "sigmoid"]


@pytest.fixture(scope="module")
def gn(gpu):
    import gn_bwd
    gn_bwd.lib()
    return gn_bwd


def rand(seed, *shape, dtype=BF, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def near(got, ref, size):
    e = torch.finfo(got.dtype).eps / 2
    d = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    bad = d > e * ref.abs() + size + torch.finfo(got.dtype).tiny
    assert not bool(bad.any()), (float((d / (e * ref.abs() + size + 1e-300)).max()), int(bad.sum()))


def act64(x, kind):
    import torch.nn.functional as F
    return dict(none=lambda v: v, relu=torch.relu, gelu_tanh=lambda v: F.gelu(v, approximate="tanh"), gelu_erf=F.gelu,
                silu=F.silu, tanh=torch.tanh, sigmoid=torch.sigmoid)[kind](x)


def slope64(p, kind):
    """The derivative at what the backward reads."""
    if kind == "tanh":
        return 1 - p * p
    if kind == "sigmoid":
        return p * (1 - p)
    x = p.clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(x, kind).sum(), x)[0]


def product(a, b):
    """a b^T in fp64 and the fp32 product's error."""
    k = a.shape[1]
    return a.double() @ b.double().t(), 2 ** -23 * (k ** 0.5 + 8) * (a.double().abs() @ b.double().abs().t())


def check_fwd(gn, M, N, K, act="none", res=None, dtype=BF, bias=True, pre=True, inplace=False, shift=0, seed=0):
    def put(t):  # an address that no 16-byte piece starts at
        return t if not shift else torch.cat((t.new_zeros(shift), t.reshape(-1)))[shift:].view(t.shape)

    X, W = put(rand(seed, M, K, dtype=dtype)), put(rand(seed + 1, N, K, dtype=dtype, std=max(K, 1) ** -0.5))
    b = put(rand(seed + 2, N, dtype=dtype)) if bias else None
    R = None if res is None else put(rand(seed + 3, M, N, dtype=res))
    r64 = 0 if R is None else R.double()
    got = gn.linear_act_fwd(X, W, b, act=act, residual=R, need_pre=pre, out=R if inplace else None)
    Y, P = got if pre else (got, None)
    if inplace:
        assert Y is R
    assert Y.dtype is (res or dtype)
    v, e = product(X, W)
    if bias:
        v = v + b.double()
        e = e + 2 ** -23 * v.abs()
    a = act64(v, act)
    ea = e if act in ("none", "relu") else 1.13 * e + 2 ** -20 * (1 + v.abs())
    if pre:
        assert P.dtype is dtype
        near(P, *((a, ea) if act in ("tanh", "sigmoid") else (v, e)))
    near(Y, a + r64, ea + 2 ** -23 * (a + r64).abs())


def check_bwd(gn, M, N, K, act, dtype=BF, shift=0, seed=0, accumulate=False, inplace=False):
    def put(t):
        return t if not shift else torch.cat((t.new_zeros(shift), t.reshape(-1)))[shift:].view(t.shape)

    dY, W, P = rand(seed, M, N, dtype=dtype, std=0.01), rand(seed + 1, N, K, dtype=dtype, std=0.05), rand(seed + 2, M, K, dtype=dtype)
    A = act64(P.double(), act).to(dtype)
    P = A.clone() if act in ("tanh", "sigmoid") else P
    dY, W, P, A = put(dY), put(W), put(P), put(A)
    p64 = P.double()
    kw = {}
    add_w = add_b = 0
    if accumulate:
        kw = dict(dW=rand(seed + 5, N, K, dtype=F32), db=rand(seed + 6, N, dtype=F32), accumulate=True)
        add_w, add_b = kw["dW"].double(), kw["db"].double()
    if inplace:
        kw["dP"] = P
    dP, dW, db = gn.act_linear_bwd(act, dY, P, A, W, **kw)
    v, e = product(dY, W.t())
    s = slope64(p64, act)
    es = 0 if act in ("relu", "tanh", "sigmoid") else 2 ** -19 * (1 + p64.abs())
    near(dP, v * s, e * s.abs() + v.abs() * (es + 2 ** -22))
    v, e = product(dY.t(), A.t())
    near(dW, v + add_w, e + 2 ** -23 * abs(add_w))
    near(db, dY.double().sum(0) + add_b, 2 ** -23 * (M ** 0.5 + 8) * dY.double().abs().sum(0) + 2 ** -23 * abs(add_b))


@pytest.mark.parametrize("act", ["none"] + ACTS)
@pytest.mark.parametrize("dtype,res", [(BF, None), (BF, BF), (BF, F32), (F32, None), (F32, F32)])
def test_forward_kinds(gn, act, dtype, res):
    for M, N, K in ((3, 40, 64), (70, 200, 136), (260, 264, 72)):
        for pre in (False, True):
            check_fwd(gn, M, N, K, act, res, dtype, pre=pre)
    check_fwd(gn, 33, 64, 32, act, res, dtype, bias=False)


# sizes of every kernel: small tiles (32 and 64 a side), 128- and 256-row streamed tiles, more than one tile a block
SIZES = [(1, 8, 8), (1, 5632, 2048), (8, 5632, 2048), (64, 2048, 5632), (130, 1000, 64), (384, 768, 768), (1003, 2304, 768),
         (2048, 2048, 256), (4001, 5632, 136), (8190, 768, 768), (5000, 4096, 64)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_sizes(gn, M, N, K):
    check_fwd(gn, M, N, K, "gelu_tanh", None)
    check_fwd(gn, M, N, K, "none", F32, pre=False)
    check_fwd(gn, M, N, K, "silu", BF, pre=False)


ODD = [(1, 1, 1), (5, 7, 9), (1, 33, 100), (65, 129, 67), (300, 1001, 203), (1000, 999, 1003), (4099, 1025, 333), (7, 8, 513), (40, 36, 64)]


@pytest.mark.parametrize("M,N,K", ODD)
def test_odd_sizes(gn, M, N, K):
    for dtype in (BF, F32):
        check_fwd(gn, M, N, K, "gelu_erf", F32, dtype)
        check_fwd(gn, M, N, K, "none", dtype, dtype, pre=False)
        check_bwd(gn, M, N, K, "silu", dtype)


@pytest.mark.parametrize("shift", [1, 4])
def test_unaligned_views(gn, shift):
    for M, N, K in ((20, 64, 64), (700, 1024, 256), (33, 50, 40)):
        check_fwd(gn, M, N, K, "silu", BF, shift=shift)
        check_fwd(gn, M, N, K, "relu", F32, shift=shift)
        check_bwd(gn, M, N, K, "gelu_tanh", shift=shift)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_backward_kinds(gn, act, dtype):
    for M, N, K in ((5, 40, 64), (300, 136, 264), (1100, 768, 512)):
        check_bwd(gn, M, N, K, act, dtype)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_backward_sizes(gn, M, N, K):
    check_bwd(gn, M, N, K, "gelu_tanh")


def test_in_place_and_accumulate(gn):
    for M, N, K in ((9, 40, 64), (600, 512, 256), (50, 63, 77)):
        check_fwd(gn, M, N, K, "none", F32, BF, inplace=True, pre=False)
        check_fwd(gn, M, N, K, "silu", BF, BF, inplace=True)
        check_fwd(gn, M, N, K, "silu", F32, F32, inplace=True)
        check_bwd(gn, M, N, K, "silu", accumulate=True, inplace=True)
        check_bwd(gn, M, N, K, "silu", F32, accumulate=True)


def test_parts_left_out(gn):
    M, N, K = 300, 128, 256
    dY, P, W = rand(1, M, N), rand(2, M, K), rand(3, N, K)
    A = act64(P.double(), "silu").to(BF)
    full = gn.act_linear_bwd("silu", dY, P, A, W)
    only = gn.act_linear_bwd("silu", dY, P, None, W, need_dw=False)
    assert torch.equal(only[0], full[0]) and only[1:] == (None, None)
    only = gn.act_linear_bwd("silu", dY, None, A, W, need_dp=False)
    assert only[0] is None and torch.equal(only[1], full[1]) and torch.equal(only[2], full[2])
    only = gn.act_linear_bwd("silu", dY, P, A, W, need_db=False)
    assert only[2] is None
    near(only[1], full[1].double(), 2 ** -20 * (dY.double().abs().t() @ A.double().abs()))


def test_empty_sizes(gn):
    X, W, b, R = rand(1, 5, 0), rand(2, 6, 0), rand(3, 6), rand(4, 5, 6, dtype=F32)
    Y, P = gn.linear_act_fwd(X, W, b, act="relu", residual=R, need_pre=True)
    assert torch.equal(P, b.expand(5, 6)) and torch.equal(Y, R + torch.relu(b.float()))
    assert gn.linear_act_fwd(rand(1, 0, 8), rand(2, 6, 8), b).shape == (0, 6)
    dP, dW, db = gn.act_linear_bwd("relu", rand(1, 0, 6), rand(1, 0, 8), rand(1, 0, 8), rand(2, 6, 8))
    assert dP.shape == (0, 8) and float(dW.abs().max()) == float(db.abs().max()) == 0
    dP, dW, db = gn.act_linear_bwd("relu", rand(1, 4, 0), rand(1, 4, 8), rand(1, 4, 8), rand(2, 0, 8))
    assert float(dP.abs().max()) == 0 and dW.shape == (0, 8)


def test_extreme_arguments(gn):
    """Large pre-activations saturate without NaN: W is the unit matrix, so v is X itself."""
    x = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 20., -20., 90., -90., 200., -200., 3e4, -3e4, 3e38, -3e38, 1e-38, -1e-38], device=DEV)
    for dtype in (BF, F32):
        X = x.to(dtype).view(16, 1) * torch.eye(16, device=DEV, dtype=dtype)[:1]
        W = torch.eye(16, device=DEV, dtype=dtype)[:, :16].contiguous()
        for act in ACTS:
            near(gn.linear_act_fwd(X.contiguous(), W, act=act), act64(X.double(), act),
                 2 ** -20 * (1 + X.double().abs().clamp(max=128)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu_tanh", "gelu_erf"])
def test_small_arguments(gn, act, dtype):
    """Towards 0 an activation is good to a part of itself, not of 1: its terms of x have at most 2^-20 of themselves as error, and tanh
    from 0.245 on 2^-22 of 1 (W is the unit matrix)."""
    x = torch.tensor([1e-30, -1e-20, 1e-10, 1e-7, -1e-6, 1e-5, 1e-4, -1e-3, 0.01, 0.06, -0.1, 0.2, 0.249, 0.251, -0.3, 0.5], device=DEV)
    X = x.to(dtype).view(1, 16).repeat(16, 1)
    Y = gn.linear_act_fwd(X, torch.eye(16, device=DEV, dtype=dtype), act=act)
    ref = act64(X.double(), act)
    near(Y, ref, 2 ** -19 * ref.abs())


def test_extreme_slopes(gn):
    """Derivatives far from 0: those of the activations' ends, and no NaN (W is the unit matrix: dP = dY act'(P))."""
    x = torch.tensor([0.0, 5., -5., 19., -19., 21., -21., 90., -90., 1e4, -1e4, 1e20, -1e20, 1e30, -1e30, 1e-30], device=DEV)
    for dtype in (BF, F32):
        P = x.to(dtype).view(1, 16).repeat(16, 1)
        W = torch.eye(16, device=DEV, dtype=dtype)
        dY = torch.ones(16, 16, device=DEV, dtype=dtype)
        for act in ("relu", "gelu_tanh", "gelu_erf", "silu"):
            p = P.double().clamp(-600, 600)  # fp64's own 0 times inf
            dP = gn.act_linear_bwd(act, dY, P, None, W, need_dw=False)[0]
            near(dP, slope64(p, act), 2 ** -19 * (1 + p.abs()).clamp(max=128))


def test_rows_as_long_as_they_may_be(gn):
    """Rows of 2^23 - 8 elements: a tile's last ones begin 2^32 bytes behind its first, less some.  Whole numbers in four columns,
    0 elsewhere: every sum is exact."""
    M, K, L = 512, 512, 2 ** 23 - 8
    cols = [0, 5, L // 2 + 3, L - 1]
    small = torch.randint(-3, 4, (M, 4), device=DEV).to(BF), torch.randint(-3, 4, (K, 4), device=DEV).to(BF)

    def long(t):
        out = torch.zeros(len(t), L, dtype=BF, device=DEV)
        out[:, cols] = t
        return out

    X, W = long(small[0]), long(small[1])
    want = small[0].double() @ small[1].double().T
    assert torch.equal(gn.linear_act_fwd(X, W, act="relu").double(), want.clamp(min=0))
    del W
    K = 128
    P, A = torch.ones(M, K, dtype=BF, device=DEV), torch.randint(-3, 4, (M, K), device=DEV).to(BF)
    W = torch.zeros(L, K, dtype=BF, device=DEV)
    W[cols] = small[1][:K].T.contiguous()
    dP, dW, db = gn.act_linear_bwd("relu", X, P, A, W)
    assert torch.equal(dP.double(), want[:, :K])
    assert torch.equal(dW[cols].double(), small[0].double().T @ A.double()) and torch.equal(db[cols].double(), small[0].double().sum(0))
    dW[cols] = 0
    assert not bool(dW.any()) and int(db.count_nonzero()) <= 4


def test_elements_past_31_bits(gn):
    """Outputs, residuals and stored sums of more than 2^31 elements, of small whole numbers: every sum is exact."""
    M, N, K = 270001, 8008, 16
    whole = lambda *shape: torch.randint(-3, 4, shape, device=DEV, dtype=torch.int8).to(BF)  # noqa: E731
    X, W, R = whole(M, K), whole(N, K), whole(M, N)
    Y, P = gn.linear_act_fwd(X, W, act="relu", residual=R, need_pre=True)
    rows = [0, 1, M // 2, M - 300, M - 1]
    v = X[rows].double() @ W.double().T
    assert torch.equal(P[rows].double(), v) and torch.equal(Y[rows].double(), v.clamp(min=0) + R[rows].double())
    dY, W2 = whole(M, K), whole(K, N)
    dP, dW, db = gn.act_linear_bwd("relu", dY, P, R, W2, dP=Y)
    assert torch.equal(dP[rows].double(), dY[rows].double() @ W2.double() * (P[rows] > 0))
    at = [0, 3, N // 2, N - 1]
    assert torch.equal(dW[:, at].double(), dY.double().T @ R[:, at].double()) and torch.equal(db.double(), dY.double().sum(0))


def test_a_block_of_both(gn):
    """The feed-forward block as it is trained: up with its activation, down with the fp32 residual, and back, against
    autograd in fp64 at the saved tensors."""
    T, d, ff = 520, 256, 1024
    x, stream = rand(1, T, d), rand(2, T, d, dtype=F32)
    W1, b1, W2, b2 = rand(3, ff, d, std=d ** -0.5), rand(4, ff), rand(5, d, ff, std=ff ** -0.5), rand(6, d)
    A, P = gn.linear_act_fwd(x, W1, b1, act="gelu_tanh", need_pre=True)
    y = gn.linear_act_fwd(A, W2, b2, residual=stream)
    v, e = product(A, W2)
    near(y, v + b2.double() + stream.double(), e + 2 ** -22 * (v.abs() + b2.double().abs() + stream.double().abs()))
    dy = rand(7, T, d, std=0.01)
    dP, dW2, db2 = gn.act_linear_bwd("gelu_tanh", dy, P, A, W2)
    dx, dW1, db1 = gn.linear_bwd(dP, x, W1)
    ref = (dy.double() @ W2.double()) * slope64(P.double(), "gelu_tanh")
    assert float((dP.double() - ref).norm() / ref.norm()) < 2 ** -8
    rx = ref @ W1.double()
    # dP's rounding, half a step in random directions, and dx's own
    assert float((dx.double() - rx).norm() / rx.norm()) < 2 ** -7
    assert float((dW1.double() - ref.t() @ x.double()).norm() / (ref.t() @ x.double()).norm()) < 2 ** -8


def test_gradient_against_differences(gn):
    """dP in fp32 against differences of the forward of act and the layer behind it."""
    M, N, K = 12, 24, 20
    P, W, c = rand(1, M, K, dtype=F32), rand(2, N, K, dtype=F32, std=0.3), rand(3, M, N, dtype=F32)
    I = torch.eye(K, device=DEV)
    for act in ACTS[1:]:
        A = gn.linear_act_fwd(P, I, act=act)
        saved = A if act in ("tanh", "sigmoid") else P
        dP, dW, db = gn.act_linear_bwd(act, c, saved, A, W)
        v = rand(4, M, K, dtype=F32)
        f = lambda e: float((gn.linear_act_fwd(gn.linear_act_fwd(P + e * v, I, act=act), W).double() * c.double()).sum())  # noqa: E731
        e = 2.0 ** -5
        slope = (8 * (f(e) - f(-e)) - (f(2 * e) - f(-2 * e))) / (12 * e)
        size = float((dP.double() * v.double()).abs().sum())
        # e^4 / 30 of a fifth derivative of up to 30 or so times v^5, and the forward's roundings over e
        assert abs(slope - float((dP.double() * v.double()).sum())) < 2 ** -9 * size + 2 ** -18 * (M * N * K) ** 0.5 / e, act


def test_another_stream_two_at_once_and_replays(gn):
    M, N, K = 1000, 768, 520
    X, W, b, R = rand(1, M, K), rand(2, N, K, std=0.05), rand(3, N), rand(4, M, N, dtype=F32)
    dY, P = rand(5, M, N), rand(6, M, K)
    A = act64(P.double(), "silu").to(BF)
    ref = gn.linear_act_fwd(X, W, b, act="silu", residual=R, need_pre=True)
    back = gn.act_linear_bwd("silu", dY, P, A, W)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(gn.linear_act_fwd(X, W, b, act="silu", residual=R, need_pre=True) + gn.act_linear_bwd("silu", dY, P, A, W))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(u, v) for u, v in zip(g, ref + back))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gn.linear_act_fwd(X, W, b, act="silu", residual=R, need_pre=True) + gn.act_linear_bwd("silu", dY, P, A, W)
    for k in range(4):
        X.copy_(rand(10 + k, M, K))
        dY.copy_(rand(20 + k, M, N))
        graph.replay()
        torch.cuda.synchronize()
        want = gn.linear_act_fwd(X, W, b, act="silu", residual=R, need_pre=True) + gn.act_linear_bwd("silu", dY, P, A, W)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(y, want))
