"""What linear_act_fwd and act_linear_bwd refuse, before any HIP call (no GPU needed)."""
import os

import pytest

gn = pytest.importorskip("gn_bwd")
if not os.path.exists(gn.LIB_PATH):
    pytest.skip("libgn_bwd.so not built", allow_module_level=True)

BASE, MB = 1 << 30, 1 << 20  # addresses that are never read: the checks come first
X, W, B, R, P, Y, A, DP, DW, DB, WS = (BASE + k * MB for k in range(11))
M, N, K = 16, 64, 32


def refused(rc, text, code=-1):
    assert rc == code and text in gn.last_error(), (rc, gn.last_error())


def fwd(act=3, x=X, w=W, b=B, r=R, p=P, y=Y, m=M, n=N, k=K, dt=gn.BF16, yd=gn.F32, ws=None, nb=0):
    return gn.lib().gn_linear_act_fwd(act, x, w, b, r, p, y, m, n, k, dt, yd, ws, nb, None)


def bwd(act=3, dy=Y, p=P, a=A, w=W, dp=DP, dw=DW, db=DB, m=M, n=N, k=K, dt=gn.BF16, ws=None, nb=0):
    return gn.lib().gn_act_linear_bwd(act, dy, p, a, w, dp, dw, db, m, n, k, dt, 0, ws, nb, None)


@pytest.mark.parametrize("call", [fwd, bwd])
def test_both_refuse(call):
    refused(call(m=-1), "negative")
    refused(call(dt=gn.F16), "dtype")
    refused(call(m=1 << 28), "2^28")
    refused(call(n=1 << 23), "2^23")
    refused(call(k=1 << 23), "2^23")
    refused(call(m=1 << 20, n=1 << 16), "2^36")
    refused(call(n=1 << 20, k=1 << 16), "2^36")
    refused(call(act=6), "activation")
    refused(call(w=None), "null")
    refused(call(w=W + 1), "aligned")
    refused(call(p=P + 1), "aligned")
    refused(call(w=W + 2), "workspace", -3)  # not in 16-byte pieces
    refused(call(k=33), "workspace", -3)
    need = gn.linear_act_workspace_bytes(M, N, 33, gn.BF16)
    refused(call(k=33, ws=WS + 8, nb=need), "workspace", -3)
    refused(call(k=33, ws=WS, nb=16), "workspace", -3)


def test_forward_refuses():
    refused(fwd(act=-2), "activation")
    refused(fwd(dt=gn.F32, yd=gn.BF16), "y dtype")
    refused(fwd(yd=gn.F16), "y dtype")
    refused(fwd(x=None), "null")
    refused(fwd(y=None), "null")
    refused(fwd(y=Y + 2), "aligned")
    refused(fwd(b=B + 1), "aligned")
    refused(fwd(y=R + 4), "share memory")
    refused(fwd(y=X), "share memory")
    refused(fwd(y=W), "share memory")
    refused(fwd(p=Y), "share memory")
    refused(fwd(p=R), "share memory")
    refused(fwd(k=33, ws=Y, nb=1 << 16), "share memory")
    refused(fwd(dt=gn.F32, y=R, p=None), "only with P")


def test_backward_refuses():
    refused(bwd(act=-1), "activation")
    refused(bwd(dy=None), "null")
    refused(bwd(p=None), "null")
    refused(bwd(a=None), "null")
    refused(bwd(dw=None), "db without dW")
    refused(bwd(dw=DW + 2), "aligned")
    refused(bwd(dp=P, a=P), "share memory")
    refused(bwd(dp=P + 16), "share memory")
    refused(bwd(dp=P, dt=gn.F32), "fp32 dP")
    refused(bwd(dp=Y), "share memory")
    refused(bwd(dw=A), "share memory")
    refused(bwd(db=DW + 64), "share memory")
    refused(bwd(ws=DP, nb=64), "share memory")


def test_workspace_query():
    q = gn.lib().gn_linear_act_workspace_bytes
    assert q(8, 8, 8, gn.F32) == q(0, 8, 8, gn.BF16) == q(8, 8, 1 << 28, gn.BF16) == q(8, 8, 8, gn.F16) == 0
    assert q(3, 5, 7, gn.BF16) >= (3 * 8 + 8 * 8) * 2


def test_nothing_to_do():
    assert fwd(m=0) == 0 and fwd(n=0) == 0
    assert bwd(m=0, dp=None, dw=None, db=None) == 0
