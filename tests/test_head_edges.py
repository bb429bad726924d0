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
