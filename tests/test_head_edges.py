"""What rope, qk_norm_rope, linear_xent and their neighbours refuse at their borders, before any HIP
call (no GPU needed)."""
import ctypes
import os

import pytest

gn = pytest.importorskip("gn_bwd")
if not os.path.exists(gn.LIB_PATH):
    pytest.skip("libgn_bwd.so not built", allow_module_level=True)

BASE = 1 << 30  # addresses that are never read: the checks come first
MB = 1 << 20


def p(off=0):
    return ctypes.c_void_p(BASE + off)


def refused(rc, text, code=-1):
    assert rc == code and text in gn.last_error(), (rc, gn.last_error())


@pytest.mark.parametrize("T,d,V", [(1 << 23, 8, 1 << 20), (1 << 27, 8, 1 << 16), (1 << 22, 1 << 20, 1 << 20)])
def test_more_tiles_than_a_product_counts(T, d, V):
    lib = gn.lib()
    refused(lib.gn_linear_xent_fwd(p(), p(), p(), p(), None, T, d, V, 4, p(), 1, None), "2^43")
    refused(lib.gn_linear_xent_bwd(p(), p(), p(), p(), None, None, 1.0, p(), p(), 0, T, d, V, 4, 0, p(), 1, None), "2^43")


def test_nodes_check_their_tensors():
    """Sizes and types by which a node's backward would read or write past its tensors."""
    gc = pytest.importorskip("grilly_core")
    import grilly_bridge as gb
    op, F, H = gc.OpType, gb.DTYPE_F32, gb.DTYPE_BF16
    ref = lambda dtype, *shape: gb.make_tensor_ref(BASE, shape, dtype, True)
    q, k = ref(H, 2, 4, 64, 32), ref(H, 2, 2, 64, 32)

    def bad(match, *args):
        with pytest.raises(ValueError, match=match):
            gc._check_node(*args)

    # attention: fewer key and value heads than query heads, another type, no V
    gc._check_node(op.FlashAttention2, [q, q, q], [q])
    gc._check_node(op.FlashAttention2, [q, q, q, ref(F, 2, 64)], [q])
    bad("repeated", op.FlashAttention2, [q, k, k], [q])
    bad("repeated", op.FlashAttention2, [q, q, k], [q])
    bad("repeated", op.FlashAttention2, [q, q, ref(F, 2, 4, 64, 32)], [q])
    bad("repeated", op.FlashAttention2, [q, q, q], [k])
    bad("repeated", op.FlashAttention2, [q, q], [q])
    fused = gb.attention_params(fused_qkv_heads=4)
    gc._check_node(op.FlashAttention2, [ref(H, 2, 64, 384)], [ref(H, 2, 64, 128)], fused)
    bad("third", op.FlashAttention2, [ref(H, 2, 64, 384)], [ref(H, 3, 64, 128)], fused)
    bad("third", op.FlashAttention2, [ref(H, 2, 64, 384)], [ref(F, 2, 64, 128)], fused)
    # rotation and norms: a gradient of the output's type is read by the input's
    x = ref(F, 2, 8, 256)
    for o in (op.Rope, op.QkNormRope):
        gc._check_node(o, [x], [x])
        bad("type", o, [x], [ref(H, 2, 8, 256)])
    # the loss: a gradient per row is read
    h, t, loss = ref(H, 16, 64), ref(3, 16), ref(F, 16)
    gc._check_node(op.LinearCrossEntropy, [h, t], [loss], b"", True)
    gc._check_node(op.LinearCrossEntropy, [h, t], [ref(F, 1)], b"", False)
    bad("upstream", op.LinearCrossEntropy, [h, t], [ref(F, 1)], b"", True)
    bad("upstream", op.LinearCrossEntropy, [h, t], [ref(H, 16)], b"", True)


def test_attention_takes_one_size():
    """K and V of fewer heads than Q would be read past their end."""
    torch = pytest.importorskip("torch")
    q, k = torch.zeros(2, 4, 64, 32), torch.zeros(2, 2, 64, 32)
    lse = torch.zeros(2, 4, 64)
    for args in ((k, k), (q, k), (k, q), (q.bfloat16(), q), (q[:, :, :32], q)):
        with pytest.raises(gn.GnError, match="as Q"):
            gn.attn_fwd(q, *args)
        with pytest.raises(gn.GnError, match="as Q"):
            gn.attn_bwd(q, *args, q, q, lse)
    with pytest.raises(gn.GnError, match="repeated"):
        gn.attn_fwd(q, k, k)
    with pytest.raises(gn.GnError, match="as Q"):
        gn.attn_bwd(q, q, q, q, k, lse)
    with pytest.raises(gn.GnError, match="as Q"):
        gn.attn_bwd(q, q, q, q, q, lse, out=(q, k, q))
    with pytest.raises(gn.GnError, match="not on the GPU"):  # of one size: on to the next check
        gn.attn_fwd(q, q, q)


B, S, D = 2, 8, 64


def heads(off=0, H=2, sb=None, ss=None, sh=None):
    ss = H * D if ss is None else ss
    return gn.Heads(BASE + off, S * ss if sb is None else sb, ss, D if sh is None else sh, H)


def turn(**kw):
    r = gn.Rope(BASE >> 1, None, 0, 0, 1.0, D, 2)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def test_rope_output_over_its_tables():
    """An output may not lie over the frequencies or the positions (rows of 128 bytes a head, 4096 in all)."""
    for fn in (gn.lib().gn_rope_fwd, gn.lib().gn_rope_bwd):
        for off in (-248, 0, 100 * 8, 4088):
            refused(fn(heads(), heads(MB), turn(freqs=BASE + MB + off), B, S, D, 4, None), "freqs")
        refused(fn(heads(), heads(), turn(positions=BASE + 4092), B, S, D, 4, None), "positions")
        refused(fn(heads(), heads(MB), turn(positions=BASE + MB - 36, pos_sb=2), B, S, D, 4, None), "positions")
        # a table between an output's heads, and into the next one by its last 8 bytes
        far = heads(MB, sb=64 * S * D, ss=64 * D, sh=32 * D)
        refused(fn(heads(), far, turn(freqs=BASE + MB + 33 * 128 - 248 + 31 * 128), B, S, D, 4, None), "freqs")


def test_qk_weight_gradients_and_workspace_stand_alone():
    lib = gn.lib()
    q, k, dyq, dyk, dyv = (heads(i * MB) for i in range(5))
    dq, dk, dv = (heads(i * MB) for i in range(5, 8))
    w, ws = p(8 * MB), p(9 * MB)
    dw = [p(10 * MB), p(11 * MB)]

    def bwd(dwq=dw[0], dwk=dw[1], ws=ws, wq=w, r=turn()):
        return lib.gn_qk_norm_rope_bwd(dyq, dyk, dyv, q, k, wq, w, dq, dk, dv, dwq, dwk, r, B, S, D, 1e-6, 4, 0, ws, 1 << 20,
                                       None)

    for i in range(8):
        refused(bwd(dwq=p(i * MB)), "shares memory")
        refused(bwd(dwk=p(i * MB + 4096 - 4)), "shares memory")
        refused(bwd(ws=p(i * MB + 4096 - 16)), "shares memory")
    refused(bwd(dwq=p(8 * MB + 124)), "may not share")     # the weights' last bytes
    refused(bwd(dwk=p(9 * MB)), "may not share")           # the workspace
    refused(bwd(r=turn(freqs=BASE + 9 * MB)), "may not share")
    refused(bwd(dwq=w), "may not share")
    refused(bwd(wq=p(5 * MB + 16)), "dq shares memory with wq")

    def fwd(wq=w, wk=w, r=turn()):
        return lib.gn_qk_norm_rope_fwd(q, k, dyv, wq, wk, dq, dk, dv, r, B, S, D, 1e-6, 4, None)

    refused(fwd(wq=p(6 * MB)), "yk shares memory with wq")
    refused(fwd(wk=p(7 * MB + 4094)), "yv shares memory with wk")
    refused(fwd(r=turn(freqs=BASE + 5 * MB)), "yq shares memory with freqs")


def test_between_the_heads_is_free():
    """A weight gradient in the gap between the parts of fused rows touches none of them: on to the check of
    the workspace; one element further it is refused."""
    lib = gn.lib()
    C = 1024  # q, k, v of two heads, then 640 elements of something else
    part = lambda off, i: gn.Heads(BASE + off + i * 2 * D * 2, S * C, C, D, 2)
    d = [part(MB, i) for i in range(3)]
    dy = [heads((3 + i) * MB) for i in range(3)]
    gap = BASE + MB + 3 * C * 2 + 6 * D * 2  # behind row 3's heads

    def go(dwq, ws, wsb=1 << 20):
        return lib.gn_qk_norm_rope_bwd(dy[0], dy[1], dy[2], part(0, 0), part(0, 1), None, None, *d, ctypes.c_void_p(dwq), None,
                                       turn(), B, S, D, 1e-6, 4, 0, ws, wsb, None)

    refused(go(gap, None, 0), "workspace", -3)
    refused(go(gap, p(4 * MB)), "the workspace shares memory with dyk")  # dwq itself passed
    refused(go(gap - 4, p(9 * MB)), "dv shares memory with dwq")
    refused(go(gap + 640 * 2 - 4 * D + 4, p(9 * MB)), "dq shares memory with dwq")


def test_linear_xent_outputs_and_workspace_stand_alone():
    lib = gn.lib()
    T, d, V = 16, 64, 100
    need = lib.gn_linear_xent_workspace_bytes(T, d, V, 4)
    GB = 1 << 30

    def fwd(loss=p(3 * MB), lse=p(4 * MB), ws=p(GB)):
        return lib.gn_linear_xent_fwd(p(), p(MB), p(2 * MB), loss, lse, T, d, V, 4, ws, need, None)

    last = {0: T * d * 2, 1: V * d * 2, 2: T * 4}  # bytes of h, E, targets
    for i, n in last.items():
        refused(fwd(loss=p(i * MB + n - 4)), "loss and")
        refused(fwd(lse=p(i * MB)), "lse and")
        refused(fwd(ws=p(i * MB)), "workspace")
        refused(fwd(ws=p(i * MB + n - 16)), "may not share")
    refused(fwd(ws=p(3 * MB)), "loss and the workspace")
    refused(fwd(lse=p(GB)), "lse and the workspace")

    def bwd(lse=p(3 * MB), dloss=p(4 * MB), dlse=p(5 * MB), dh=p(6 * MB), dE=p(7 * MB), ws=p(GB)):
        return lib.gn_linear_xent_bwd(p(), p(MB), p(2 * MB), lse, dloss, dlse, 1.0, dh, dE, 0, T, d, V, 4, 0, ws, need, None)

    last.update({3: T * 4, 4: T * 4, 5: T * 4})
    for i, n in last.items():
        refused(bwd(dh=p(i * MB + n - 4)), "dh and")
        refused(bwd(dE=p(i * MB + n - 4)), "dE and")
        refused(bwd(ws=p(i * MB)), "may not share")
    refused(bwd(ws=p(7 * MB + V * d * 4 - 16)), "dE and the workspace")
    refused(bwd(ws=p(6 * MB)), "dh and the workspace")


def test_sizes_past_31_bits():
    """Sizes that the entries' ints would cut off: [2^32 + 2, ...] is not [2, ...]."""
    torch = pytest.importorskip("torch")
    n = 2 ** 32 + 2
    long = torch.zeros(1).expand(n, 1)
    short, t = torch.zeros(2, 1), torch.zeros(2, dtype=torch.int32)
    for h, E in ((long, short), (short, long), (long.t(), long.t())):
        with pytest.raises(gn.GnError, match="31 bits"):
            gn.linear_xent_fwd(h, E, t)
        with pytest.raises(gn.GnError, match="31 bits"):
            gn.linear_xent_bwd(h, E, t, t)
    with pytest.raises(gn.GnError, match="31 bits"):
        gn._int32("x", torch.zeros(1, 1, 1, 2).expand(n, 1, 1, 2))
    with pytest.raises(gn.GnError, match="64 bits"):
        gn._rope(torch.ones(4, dtype=torch.float64), "half", None, 2 ** 64 + 5, 1.0, 1, 1)


@pytest.mark.parametrize("dtype", [0, 4])
def test_workspace_query_of_refused_sizes(dtype):
    """0, as for other sizes that are not taken (rounding 2^31 - 1 up overflowed)."""
    top = 2 ** 31 - 1
    for size in ((top, 8, 8), (8, top, 8), (8, 8, top), (1 << 28, 8, 8), (8, (1 << 20) + 1, 8), (8, 8, 1 << 30),
                 (1 << 23, 8, 1 << 20)):
        assert gn.lib().gn_linear_xent_workspace_bytes(*size, dtype) == 0
    assert gn.lib().gn_linear_xent_workspace_bytes((1 << 28) - 1, 8, 100, dtype) > 0
    assert gn.lib().gn_linear_xent_workspace_bytes(8, 1 << 20, (1 << 30) - 1, dtype) > 0


def test_default_eps_of_the_parameter_blocks():
    """1e-6 where the block has key and value heads, whichever helper packs it; a given 0 stays 0."""
    import struct
    pytest.importorskip("grilly_core")
    import grilly_bridge as gb
    eps = lambda block: struct.unpack("<IIIIffIi", block)[5]
    want = struct.unpack("<f", struct.pack("<f", 1e-6))[0]
    assert eps(gb.rope_params(4, 64, kv_heads=2)) == eps(gb.qk_norm_rope_params(4, 2, 64)) == want
    assert eps(gb.rope_params(4, 64, kv_heads=2, eps=0.0)) == eps(gb.qk_norm_rope_params(4, 2, 64, eps=0.0)) == 0
    assert eps(gb.rope_params(4, 64)) == 0


def test_rows_past_a_launch():
    """A block of 256 threads a row: from 2^24 rows on the grid would wrap around without an error."""
    lib = gn.lib()
    n = 1 << 24
    a, b, c, w = p(), p(1 << 40), p(2 << 40), p(3 << 40)
    for dtype in (0, 4):
        refused(lib.gn_softmax_bwd(a, b, c, n, 8, dtype, None), "rows")
        refused(lib.gn_xent_bwd(a, w, c, n, 8, 1.0, dtype, None), "rows")
        refused(lib.gn_layernorm_fwd(a, None, None, b, None, None, n, 12, 1e-5, dtype, 0, None), "rows")
        refused(lib.gn_rmsnorm_fwd(a, None, b, None, 1 << 26, 64, 1e-6, dtype, None), "rows")  # a wave a row
        refused(lib.gn_rmsnorm_bwd(a, b, w, w, c, None, n, 64, dtype, 0, None, 0, None), "rows")      # dX alone
        refused(lib.gn_rmsnorm_bwd(a, b, w, w, c, w, n, 12, dtype, 0, None, 0, None), "rows")
