"""What rope, qk_norm_rope and linear_xent refuse, before any HIP call (no GPU needed), and the
frequencies of rope_freqs."""
import ctypes
import math

import pytest

gn = pytest.importorskip("gn_bwd")
import os
if not os.path.exists(gn.LIB_PATH):
    pytest.skip("libgn_bwd.so not built", allow_module_level=True)

BASE = 1 << 30  # addresses that are never read: the checks come first
B, S, D = 2, 8, 64


def heads(off=0, H=2, sb=None, ss=None, sh=None):
    ss = H * D if ss is None else ss
    return gn.Heads(BASE + off, S * ss if sb is None else sb, ss, D if sh is None else sh, H)


def rope(**kw):
    r = gn.Rope(BASE >> 1, None, 0, 0, 1.0, D, 2)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def refused(rc, text, code=-1):
    assert rc == code and text in gn.last_error(), (rc, gn.last_error())


MB = 1 << 20


@pytest.mark.parametrize("entry", ["gn_rope_fwd", "gn_rope_bwd"])
def test_rope_refuses(entry):
    fn = getattr(gn.lib(), entry)
    x, y, r = heads(), heads(MB), rope()
    refused(fn(None, y, r, B, S, D, 4, None), "null")
    refused(fn(x, y, None, B, S, D, 4, None), "null")
    refused(fn(x, heads(MB, H=3), r, B, S, D, 4, None), "heads")
    refused(fn(x, y, r, B, S, D, 1, None), "dtype")
    refused(fn(x, y, r, B, S, 63, 4, None), "even")
    refused(fn(x, y, r, B, S, 514, 4, None), "even")
    refused(fn(x, y, r, 1 << 16, 1 << 16, D, 4, None), "2^31")
    refused(fn(x, y, rope(rot=66), B, S, D, 4, None), "rot")
    refused(fn(x, y, rope(rot=31), B, S, D, 4, None), "rot")
    refused(fn(x, y, rope(mode=0), B, S, D, 4, None), "mode")
    refused(fn(x, y, rope(freqs=None), B, S, D, 4, None), "freqs")
    refused(fn(x, y, rope(pos_sb=-1), B, S, D, 4, None), "negative")
    refused(fn(x, y, rope(freqs=BASE + 4), B, S, D, 4, None), "aligned")
    refused(fn(x, y, rope(positions=BASE + 2), B, S, D, 4, None), "aligned")
    refused(fn(x, heads(MB, ss=-1), r, B, S, D, 4, None), "negative")
    refused(fn(heads(1), y, r, B, S, D, 4, None), "aligned")
    refused(fn(heads(2), y, r, B, S, D, 0, None), "aligned")
    refused(fn(gn.Heads(None, 0, 0, 0, 2), y, r, B, S, D, 4, None), "null")
    refused(fn(heads(H=2000), heads(MB, H=2000), r, B, S, D, 4, None), "heads")
    # outputs that overlap
    refused(fn(x, heads(MB, sb=0), r, B, S, D, 4, None), "overlaps itself")
    refused(fn(x, heads(MB, sh=D - 2), r, B, S, D, 4, None), "overlaps itself")
    refused(fn(x, heads(16), r, B, S, D, 4, None), "overlaps the input")
    refused(fn(x, heads(0, sb=2 * D, ss=2 * 2 * D), r, B, S, D, 4, None), "overlaps the input")
    # nothing to do is done
    assert fn(x, y, r, 0, S, D, 4, None) == 0 and fn(x, y, r, B, 0, D, 4, None) == 0
    assert fn(heads(H=0), heads(H=0), r, B, S, D, 4, None) == 0


def test_qk_refuses():
    lib = gn.lib()
    q, k, v = heads(), heads(MB), heads(2 * MB)
    yq, yk, yv = heads(3 * MB), heads(4 * MB), heads(5 * MB)
    r = rope()
    w = ctypes.c_void_p(BASE)

    def fwd(q=q, k=k, v=v, yq=yq, yk=yk, yv=yv, r=r, eps=1e-6, dtype=4, w=w):
        return lib.gn_qk_norm_rope_fwd(q, k, v, w, w, yq, yk, yv, r, B, S, D, eps, dtype, None)

    refused(fwd(q=None), "null")
    refused(fwd(yk=None), "null")
    refused(fwd(yv=None), "null")
    refused(fwd(yq=heads(3 * MB, H=3)), "heads")
    refused(fwd(v=heads(2 * MB, H=1), yv=heads(5 * MB, H=1)), "k and v")
    refused(fwd(eps=-1.0), "eps")
    refused(fwd(eps=float("nan")), "eps")
    refused(fwd(dtype=2), "dtype")
    refused(fwd(w=ctypes.c_void_p(BASE + 1)), "weights")
    refused(fwd(yk=yq), "overlaps")
    refused(fwd(yq=k), "overlaps")       # another tensor's input
    refused(fwd(yq=heads(128)), "overlaps q")

    def bwd(dyq=yq, dyk=yk, dyv=yv, dq=heads(6 * MB), dk=heads(7 * MB), dv=heads(8 * MB), dwq=w, dwk=ctypes.c_void_p(BASE + 4 * D), flags=0,
            ws=ctypes.c_void_p(BASE), wsb=1 << 20, kk=k, S=S):
        return lib.gn_qk_norm_rope_bwd(dyq, dyk, dyv, q, kk, w, w, dq, dk, dv, dwq, dwk, r, B, S, D, 1e-6, 4, flags, ws,
                                       wsb, None)

    refused(bwd(dyq=None), "null")
    refused(bwd(dk=None), "null")
    refused(bwd(dv=None), "null")
    refused(bwd(kk=None, dyk=None, dk=None), "dwk without k")
    refused(bwd(flags=8), "flags")
    refused(bwd(dwq=ctypes.c_void_p(BASE + 2)), "aligned")
    refused(bwd(dwk=w), "share")
    refused(bwd(dwk=ctypes.c_void_p(BASE + 4 * D - 4)), "share")
    refused(bwd(dq=heads(7 * MB)), "overlaps")
    refused(bwd(ws=None, wsb=0), "workspace", -3)
    refused(bwd(wsb=64), "workspace", -3)
    refused(bwd(ws=ctypes.c_void_p(BASE + 4)), "workspace", -3)


def test_fused_rows_may_be_written_part_by_part():
    """q, k, v parts of one buffer's rows interleave without overlapping: accepted up to the
    workspace check, which comes last; one head too many is refused."""
    lib = gn.lib()
    C = 4 * D * 3
    part = lambda off, i, H=4: gn.Heads(BASE + off + i * 4 * D * 2, S * C, C, D, H)
    q, k = part(0, 0), part(0, 1)
    dy = [heads((3 + i) * MB, H=4) for i in range(3)]
    go = lambda dq: lib.gn_qk_norm_rope_bwd(dy[0], dy[1], dy[2], q, k, None, None, dq, part(MB, 1), part(MB, 2),
                                            ctypes.c_void_p(BASE), None, rope(), B, S, D, 1e-6, 4, 0, None, 0, None)
    refused(go(part(MB, 0)), "workspace", -3)
    bad = part(MB, 0)
    bad.sh = D + 2
    refused(go(bad), "overlaps")
    # heads interleaved, q and k of a head side by side: rows of [H, 3, D]
    C = 3 * 4 * D
    turn = lambda off, i: gn.Heads(BASE + off + i * D * 2, S * C, C, 3 * D, 4)
    go = lambda dq, dk: lib.gn_qk_norm_rope_bwd(dy[0], dy[1], dy[2], turn(0, 0), turn(0, 1), None, None, dq, dk,
                                                turn(MB, 2), ctypes.c_void_p(BASE), None, rope(), B, S, D, 1e-6, 4, 0,
                                                None, 0, None)
    refused(go(turn(MB, 0), turn(MB, 1)), "workspace", -3)
    refused(go(turn(MB, 0), gn.Heads(BASE + MB + D, S * C, C, 3 * D, 4)), "overlaps")


def test_linear_xent_refuses():
    lib = gn.lib()
    p = lambda off=0: ctypes.c_void_p(BASE + off)
    T, d, V = 16, 64, 100
    need = lib.gn_linear_xent_workspace_bytes(T, d, V, 4)
    assert need > 0

    def fwd(h=p(), E=p(MB), t=p(2 * MB), loss=p(3 * MB), lse=p(4 * MB), T=T, d=d, V=V, dtype=4, ws=p(5 * MB), wsb=need):
        return lib.gn_linear_xent_fwd(h, E, t, loss, lse, T, d, V, dtype, ws, wsb, None)

    refused(fwd(h=None), "null")
    refused(fwd(E=None), "null")
    refused(fwd(t=None), "null")
    refused(fwd(T=-1), "shape")
    refused(fwd(d=0), "shape")
    refused(fwd(V=0), "shape")
    refused(fwd(dtype=1), "dtype")
    refused(fwd(h=p(1)), "aligned")
    refused(fwd(t=p(2 * MB + 2)), "aligned")
    refused(fwd(loss=p(2)), "aligned")
    refused(fwd(lse=p(3 * MB)), "share")
    refused(fwd(lse=p(3 * MB + 4 * T - 4)), "share")
    refused(fwd(ws=None), "workspace", -3)
    refused(fwd(wsb=need - 1), "workspace", -3)
    refused(fwd(ws=p(5 * MB + 8)), "workspace", -3)
    assert fwd(T=0) == 0 and fwd(loss=None, lse=None) == 0

    def bwd(lse=p(3 * MB), dloss=None, dlse=None, dh=p(6 * MB), dE=p(7 * MB), ded=0, T=T, dtype=4, flags=0, ws=p(5 * MB),
            wsb=need):
        return lib.gn_linear_xent_bwd(p(), p(MB), p(2 * MB), lse, dloss, dlse, 1.0, dh, dE, ded, T, d, V, dtype, flags,
                                      ws, wsb, None)

    refused(bwd(lse=None), "null")
    refused(bwd(ded=1), "dE")
    refused(bwd(ded=4, dtype=0), "dE")
    refused(bwd(ded=4, flags=1), "accumulates")
    refused(bwd(flags=2), "flags")
    refused(bwd(dE=p(2)), "aligned")
    refused(bwd(dh=p(1)), "aligned")
    refused(bwd(dlse=p(2)), "aligned")
    refused(bwd(wsb=8), "workspace", -3)
    refused(bwd(dh=p()), "share")
    refused(bwd(dE=p(MB)), "share")
    refused(bwd(dE=p(6 * MB + 64)), "share")
    assert bwd(dh=None, dE=None) == 0 and bwd(T=0, dE=None) == 0
    for bad in ((0, 64, 100, 4), (16, 0, 100, 4), (16, 64, 0, 4), (16, 64, 100, 1)):
        assert lib.gn_linear_xent_workspace_bytes(*bad) == 0


def test_front_end_refuses():
    """The Python front end's own checks, on CPU tensors."""
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 8, 2, 64)
    f = torch.ones(32, dtype=torch.float64)
    with pytest.raises(gn.GnError, match="not on the GPU"):
        gn.rope_fwd(x, f)
    with pytest.raises(gn.GnError, match="not on the GPU"):
        gn.qk_norm_rope_fwd(x, x)
    with pytest.raises(gn.GnError, match="expected"):
        gn.linear_xent_fwd(torch.zeros(4, 8), torch.zeros(10, 9), torch.zeros(4, dtype=torch.int32))


@pytest.mark.parametrize("rot", [2, 6, 64, 128])
def test_rope_freqs(rot):
    plain = [10000.0 ** (-2 * i / rot) for i in range(rot // 2)]

    def close(a, b):
        return all(abs(x - y) <= 1e-14 * abs(y) for x, y in zip(a, b)) and len(a) == len(b)

    def get(**kw):
        f, m = gn.rope_freqs(rot, device="cpu", **kw)
        return f.tolist(), m

    f, m = get()
    assert close(f, plain) and m == 1
    assert close(get(theta=5e5)[0], [5e5 ** (-2 * i / rot) for i in range(rot // 2)])
    assert close(get(scaling="linear", factor=8.0)[0], [x / 8 for x in plain])
    f, m = get(scaling="ntk", factor=4.0)
    assert f[0] == 1 and m == 1
    if rot > 2:  # the slowest pair slows by the factor
        assert abs(f[-1] / plain[-1] * 4 - 1) < 1e-12
    f, m = get(scaling="yarn", factor=4.0, trained=2048)
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-6
    for x, y in zip(f, plain):
        turns = 2048 * y / (2 * math.pi)
        assert y / 4 * (1 - 1e-12) <= x <= y * (1 + 1e-12)
        if turns >= 32:
            assert abs(x / y - 1) < 1e-14
        if turns <= 1:
            assert abs(x * 4 / y - 1) < 1e-14


def test_rope_freqs_refuses():
    for kw in (dict(rot=3), dict(rot=-2), dict(rot=514), dict(theta=0.0), dict(theta=float("inf")),
               dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=float("nan")),
               dict(scaling="yarn", factor=2.0, trained=0), dict(scaling="yarn", factor=2.0, fast=1.0, slow=1.0)):
        with pytest.raises(gn.GnError):
            gn.rope_freqs(**{"rot": 64, "device": "cpu", **kw})


def test_node_types_and_parameters():
    """The tape's node types are appended to the numbering; their parameter blocks' layouts."""
    import struct
    grilly_core = pytest.importorskip("grilly_core")
    import grilly_bridge as gb
    assert [int(getattr(grilly_core.OpType, n)) for n in ("Embedding", "Rope", "QkNormRope", "LinearCrossEntropy")] == [
        35, 36, 37, 38]
    assert struct.unpack("<IIIIffIi", gb.rope_params(4, 32, "interleaved", 1.5, True, 7)) == (4, 0, 32, 1, 1.5, 0.0, 1, 7)
    assert struct.unpack("<IIIIffIi", gb.qk_norm_rope_params(4, 2, 64, pos0=-1))[:4] == (4, 2, 64, 2)
    assert struct.unpack("<If", gb.linear_cross_entropy_params(32000, 0.5)) == (32000, 0.5)
