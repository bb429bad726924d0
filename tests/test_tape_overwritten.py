"""What the backward of a ResidualNorm or LinearAct node reads must be as the forward left it: a node behind it that wrote the
same buffer again is refused, and nothing else is."""
import pytest

gc = pytest.importorskip("grilly_core")
import grilly_bridge as gb  # noqa: E402

F, H = gb.DTYPE_F32, gb.DTYPE_BF16
op = gc.OpType


def ref(dtype, at, *shape):
    return gb.make_tensor_ref((1 << 30) + (at << 20), shape or (6, 8), dtype, True)


def kept(*args):
    gc._check_kept(*args)


def lost(match, *args):
    with pytest.raises(ValueError, match=match):
        gc._check_kept(*args)


h, x, y, z, h2, z2, w = ref(H, 0), ref(F, 1), ref(F, 2), ref(H, 3), ref(H, 4), ref(H, 5), ref(H, 6, 8)
PRE, NONE, POST = (gb.residual_norm_params(pre="rms"), gb.residual_norm_params(), gb.residual_norm_params(post="rms"))


def test_stream_updated_in_place():
    o, none = op.ResidualNorm, [0] * 6
    again = (o, [h2, x], [x, z2])  # the next block, into the same stream
    lost("stream y", o, [h, x], [x, z], none, PRE, [again], True)
    kept(o, [h, x], [x, z], none, PRE, [again], False)  # z without a gradient: y is not read
    kept(o, [h, x], [x, z], none, PRE, [], True)  # the last block
    kept(o, [h, x], [y, z], none, PRE, [(o, [h2, y], [ref(F, 7), z2])], True)  # out of place
    lost("stream y", o, [h, x], [y, z], none, PRE, [(op.Dropout, [y], [y])], True)
    lost("stream y", o, [h, x], [y, z], none, PRE, [(op.LinearAct, [h2, y], [y]), (op.Add, [z, z2], [ref(H, 8)])], True)


def test_h_overwritten():
    o, gate = op.ResidualNorm, [0, 0, 0, 0, w.buffer_id, 0]
    again = [(op.Linear, [z], [h])]
    lost("reads h", o, [h, x], [y], [0] * 6, POST, again)
    lost("reads h", o, [h, x], [y], gate, gb.residual_norm_params(gates=1), again)
    kept(o, [h, x], [y], [0] * 6, NONE, again)  # neither norm nor gate: not read


def test_linear_act():
    o = op.LinearAct
    P = ref(H, 9)
    saved = [w.buffer_id, 0, P.buffer_id]
    act = gb.linear_act_params("silu")
    lost("reads X", o, [h], [z], saved, act, [(op.Dropout, [h], [h])])
    lost("reads P", o, [h], [z], saved, act, [(op.Linear, [z], [P])])
    kept(o, [h], [z], saved, act, [(op.Dropout, [z], [z]), (op.LinearAct, [z, y], [y])])  # its output and a stream: not read
    kept(o, [h, y], [y], [w.buffer_id, 0, 0], gb.linear_act_params(), [(op.LinearAct, [z, y], [y])])


@pytest.mark.parametrize("through", [op.Reshape, op.CubeMindSurprise, op.TemporalSurprise])
def test_a_view_overwrites_nothing(through):
    kept(op.ResidualNorm, [h, x], [y, z], [0] * 6, PRE, [(through, [y], [y])], True)
    kept(op.LinearAct, [h], [z], [w.buffer_id], gb.linear_act_params(), [(through, [h], [h])])
    lost("stream y", op.ResidualNorm, [h, x], [y, z], [0] * 6, PRE, [(through, [z], [y])], True)


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
def test_two_blocks(gpu, inplace):
    """Two pre-norm blocks whose z each has a gradient: out of place the gradients of the direct calls; with the stream in
    place the first block's y is gone, and the backward says so."""
    import numpy as np
    torch = pytest.importorskip("torch")
    import gn_bwd as gn
    dev = gc.Device(0)
    gb.attach_torch_stream(dev)
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    rows, C = 10, 64

    def rand(dtype=torch.bfloat16):
        return torch.randn(rows, C, device=gpu, generator=g).to(dtype)

    x, hs, dz = rand(torch.float32), [rand(), rand()], rand()
    w = [1 + 0.1 * rand()[0], 1 + 0.1 * rand()[1]]
    t = gb.tref
    tape = gb.create_tape_context(dev)
    tape.begin()
    stream, ys, zs = x, [], []
    for i in range(2):
        y, z = gn.residual_norm_fwd(hs[i], stream, pre="rms", pre_w=w[i], out=stream if inplace else None)
        n = tape.record_op(op.ResidualNorm, [t(hs[i], True), t(stream, True)], [t(y), t(z)], gb.residual_norm_params(pre="rms"))
        tape.save_for_backward(n, [0, 0, w[i].data_ptr()])
        stream = y
        ys.append(y)
        zs.append(z)
    out = torch.empty_like(zs[0])
    loss = tape.record_op(op.Add, [t(zs[0], True), t(zs[1], True)], [t(out)])
    if inplace:
        with pytest.raises(ValueError, match="stream y"):
            tape.backward(loss, dz.data_ptr())
        tape.end()
        return
    tape.backward(loss, dz.data_ptr())
    second = gn.residual_norm_bwd(None, dz, hs[1], ys[1], pre="rms", pre_w=w[1])
    first = gn.residual_norm_bwd(second[1], dz, hs[0], ys[0], pre="rms", pre_w=w[0])
    for v, ref_, dtype in ((x, first[1], F), (hs[0], first[0], H), (hs[1], second[0], H), (w[0], first[5], F), (w[1], second[5], F)):
        got = gb.download(dev, tape.get_grad_buffer(v.data_ptr()), v.shape, dtype)
        np.testing.assert_array_equal(got, ref_.float().cpu().numpy())
    tape.end()
