"""gn_act_bwd's slopes far from 0, which a LinearAct node takes where the layer behind it does not."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [24, 1000])
def test_gelu_slope_of_the_largest(gpu, n, dtype):
    import gn_bwd as gn
    x = torch.tensor([19.9, 20.1, 25., 1e9, 1e13, 1e19, 2e19, 1e30, 4e36, 3e38, math.inf, 5e18], device=gpu)
    x = torch.cat((x, -x)).to(dtype).repeat(n)[:n].contiguous()
    dy = torch.full_like(x, 1.5)
    assert torch.equal(gn.act_bwd("gelu_tanh", dy, x), torch.where(x > 0, 1.5, 0.0).to(dtype))
    x[1] = math.nan
    got = gn.act_bwd("gelu_tanh", dy, x)
    assert bool(torch.isnan(got[1])) and int(torch.isnan(got).sum()) == 1


def test_a_node_of_large_sums(gpu):
    """LinearAct with gelu and a pre-activation of 1e20: its slope is 1."""
    import gn_bwd as gn
    import grilly_bridge as gb
    import grilly_core as gc
    dev = gc.Device(0)
    gb.attach_torch_stream(dev)
    X = torch.tensor([[1e10, 1.0], [-1e10, 2.0]], device=gpu)
    W = torch.tensor([[1e10, 0.0], [0.0, 0.0]], device=gpu)
    dY = torch.ones(2, 2, device=gpu)
    Y, pre = gn.linear_act_fwd(X, W, act="gelu_tanh", need_pre=True)
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(gc.OpType.LinearAct, [gb.tref(X, True)], [gb.tref(Y)], gb.linear_act_params("gelu_tanh"))
    tape.save_for_backward(n, [W.data_ptr(), 0, pre.data_ptr()])
    tape.backward(n, dY.data_ptr())
    got = gb.download(dev, tape.get_grad_buffer(X.data_ptr()), X.shape, gb.DTYPE_F32)
    tape.end()
    assert abs(got[0, 0] / 1e10 - 1) < 1e-6 and got[0, 1] == 0 and got[1, 0] == 0 and got[1, 1] == 0
