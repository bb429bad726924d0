"""The tape's Dropout, ResidualNorm and LinearAct nodes: numbering, parameter blocks, and the tensors they refuse (no GPU
needed)."""
import struct

import pytest

gc = pytest.importorskip("grilly_core")
import grilly_bridge as gb  # noqa: E402

BASE = 1 << 30
F, H = gb.DTYPE_F32, gb.DTYPE_BF16
op = gc.OpType


def ref(dtype, *shape, at=0):
    return gb.make_tensor_ref(BASE + at, shape, dtype, True)


def bad(match, *args):
    with pytest.raises(ValueError, match=match):
        gc._check_node(*args)


def test_numbering_and_blocks():
    assert [int(o) for o in (op.LinearCrossEntropy, op.Dropout, op.ResidualNorm, op.LinearAct)] == [38, 39, 40, 41]
    assert struct.unpack("<dQQQ", gb.dropout_params(0.25, -1, 2, 3)) == (0.25, 2 ** 64 - 1, 2, 3)
    block = gb.residual_norm_params("rms", "layer", 4, 0.5, 2.0, 0.125, 7, 8, 9, pre_eps=1e-3)
    assert len(block) == 64
    got = struct.unpack("<dQQQffffIIIxxxx", block)
    assert got[:4] == (0.125, 7, 8, 9) and got[6:8] == (0.5, 2.0) and got[8:] == (1, 2, 4)
    assert abs(got[4] - 1e-6) < 1e-12 and abs(got[5] - 1e-3) < 1e-9
    assert struct.unpack("<i", gb.linear_act_params()) == (-1,) and struct.unpack("<i", gb.linear_act_params("silu")) == (3,)


def test_dropout_node_checks():
    gc._check_node(op.Dropout, [ref(H, 4, 8)], [ref(H, 4, 8)])
    bad("Dropout", op.Dropout, [ref(H, 4, 8)], [ref(F, 4, 8)])
    bad("Dropout", op.Dropout, [ref(H, 4, 8)], [ref(H, 4, 4)])


def test_residual_norm_node_checks():
    o = op.ResidualNorm
    h, x, y, z = ref(H, 6, 8), ref(F, 6, 8, at=1 << 20), ref(F, 6, 8, at=2 << 20), ref(H, 6, 8, at=3 << 20)
    pre, none = gb.residual_norm_params(pre="layer"), gb.residual_norm_params()
    gc._check_node(o, [h, x], [y, z], pre)
    gc._check_node(o, [h, x], [x, z], pre)  # the stream in place
    gc._check_node(o, [h, x], [y], none)
    bad("inputs h and x", o, [h], [y, z], pre)
    bad("inputs h and x", o, [h, x], [], pre)
    bad("whole block", o, [h, x], [y], none[:60])
    bad("one size", o, [h, ref(F, 6, 16)], [y, z], pre)
    bad("one size", o, [h, ref(F, 12, 4)], [y, z], pre)
    bad("one size", o, [h, x], [ref(H, 6, 8, at=2 << 20), z], pre)
    bad("z, alike h", o, [h, x], [y], pre)
    bad("z, alike h", o, [h, x], [y, z], none)
    bad("z, alike h", o, [h, x], [y, ref(F, 6, 8, at=3 << 20)], pre)
    bad("in its place", o, [h, x], [y, h], pre)
    bad("in its place", o, [ref(F, 6, 8), x], [ref(F, 6, 8)], none)


def test_linear_act_node_checks():
    o = op.LinearAct
    x, y = ref(H, 6, 8), ref(H, 6, 16)
    gc._check_node(o, [x], [y])
    gc._check_node(o, [x, ref(F, 6, 16)], [ref(F, 6, 16)])
    bad("residual's", o, [x, ref(F, 6, 16)], [y])
    bad("residual's", o, [x, ref(H, 6, 8)], [y])
    bad("f32 above", o, [ref(F, 6, 8)], [y])


def test_decoder_options():
    pytest.importorskip("torch")
    import decoder_tape
    for kw, text in ((dict(dropout=0.1), "residual_norm"), (dict(fused_linear=True, residual_norm=True), "residual sum"),
                     (dict(ffn="relu"), "ffn")):
        with pytest.raises(ValueError, match=text):
            decoder_tape.Decoder(device="cpu", **kw)
