"""What the tape's fused backward of two linear layers holds in device memory."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def held(gpu, fused, M, d, ff, shift=0):
    """Bytes that the engine's pool holds behind a backward of Linear over LinearAct; shift: elements in front of W2."""
    import gn_bwd as gn
    import grilly_bridge as gb
    import grilly_core as gc
    dev = gc.Device(0)
    gb.attach_torch_stream(dev)

    def rand(*shape):
        return torch.randn(*shape, device=gpu).to(torch.bfloat16)

    X, W1, W2, dY = rand(M, d), rand(ff, d), rand(d * ff + shift)[shift:].view(d, ff), rand(M, d)
    A, pre = gn.linear_act_fwd(X, W1, act="silu", need_pre=True)
    Y = gn.linear_act_fwd(A, W2)
    t = gb.tref
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(fused)
    tape.begin()
    n = tape.record_op(gc.OpType.LinearAct, [t(X, True)], [t(A)], gb.linear_act_params("silu"))
    tape.save_for_backward(n, [W1.data_ptr(), 0, pre.data_ptr()])
    n = tape.record_op(gc.OpType.Linear, [t(A, True)], [t(Y)])
    tape.save_for_backward(n, [W2.data_ptr()])
    tape.backward(n, dY.data_ptr())
    torch.cuda.synchronize()
    s = dev.pool_stats()
    got = gb.download(dev, tape.get_grad_buffer(X.data_ptr()), X.shape, gb.DTYPE_BF16)
    dP = gn.act_linear_bwd("silu", dY, pre, A, W2)[0]
    ref = gn.linear_bwd(dP, X, W1)[0].float().cpu().numpy()
    tape.end()
    if fused:
        assert (got == ref).all()
    return s["bytes_live"] + s["bytes_cached"]


@pytest.mark.parametrize("M,d,ff", [(1024, 768, 1024), (4096, 256, 1024)])
def test_aligned_operands_need_no_layout(gpu, M, d, ff):
    """The fused form leaves out the gradient of the activation's output and lays nothing out: it never holds more."""
    apart = held(gpu, False, M, d, ff)
    assert held(gpu, True, M, d, ff) <= apart


def test_unaligned_and_odd_operands_are_laid_out(gpu):
    held(gpu, True, 300, 264, 136, shift=1)
    held(gpu, True, 300, 263, 137)
