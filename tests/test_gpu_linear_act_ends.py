"""GPU tests of linear_act_fwd and act_linear_bwd where the numbers end: slopes of the largest P, NaN in a sum."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_linear_act import ACTS, BF, DEV, F32, near, rand  # noqa: E402


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
