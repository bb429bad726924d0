"""What dropout and residual_norm refuse, before any HIP call (no GPU needed)."""
import os

import pytest

gn = pytest.importorskip("gn_bwd")
if not os.path.exists(gn.LIB_PATH):
    pytest.skip("libgn_bwd.so not built", allow_module_level=True)

BASE, MB = 1 << 30, 1 << 20  # addresses that are never read: the checks come first


def refused(rc, text, code=-1):
    assert rc == code and text in gn.last_error(), (rc, gn.last_error())


@pytest.mark.parametrize("entry", ["gn_dropout_fwd", "gn_dropout_bwd"])
def test_dropout_refuses(entry):
    fn = getattr(gn.lib(), entry)
    tail = (0, None) if entry.endswith("bwd") else (None,)

    def call(x=BASE, y=BASE + MB, n=64, p=0.5, rng=gn.Rng(1, 2, 3), dt=gn.BF16, tail=tail):
        return fn(x, y, n, p, rng, dt, *tail)

    refused(call(n=-1), "elements")
    refused(call(n=1 << 56), "elements")
    refused(call(dt=gn.F16), "dtype")
    for p in (-0.1, 1.0, 1.5, float("nan"), 1.0 - 2.0 ** -40):
        refused(call(p=p), "p must be")
    refused(call(rng=None), "generator")
    refused(call(rng=gn.Rng(1, 2, 3, BASE + 4)), "step_dev")
    refused(call(rng=gn.Rng(1, 2, 3, BASE + MB + 8)), "step_dev")
    refused(call(x=None), "null")
    refused(call(y=None), "null")
    refused(call(x=BASE + 1), "aligned")
    refused(call(y=BASE + 2, dt=gn.F32), "aligned")
    refused(call(y=BASE + 64), "share memory")
    if entry.endswith("bwd"):
        refused(call(y=BASE, tail=(gn.ACCUMULATE, None)), "share memory")
    assert call(n=0) == 0


def branch(**kw):
    b = gn.Branch(0, 2, None, None, BASE + 8 * MB, BASE + 9 * MB, 1e-5, 1e-5, None, 0, 1.0, 1.0, 0.0)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


R, F = 6, 64
H, X, Y, Z = BASE, BASE + MB, BASE + 2 * MB, BASE + 3 * MB


def fwd(b=None, h=H, hd=gn.BF16, x=X, xd=gn.F32, y=Y, z=Z, rows=R, f=F):
    return gn.lib().gn_residual_norm_fwd(b or branch(), h, hd, x, xd, y, z, rows, f, None)


DY, DZ, DH, DX, WS, G = (BASE + k * MB for k in range(16, 22))


def bwd(b=None, dy=DY, dz=DZ, h=H, hd=gn.BF16, y=Y, xd=gn.F32, dh=DH, dx=DX, g=None, rows=R, f=F, ws=WS, nb=1 << 40):
    return gn.lib().gn_residual_norm_bwd(b or branch(), dy, dz, h, hd, y, xd, dh, dx, g, rows, f, 0, ws, nb, None)


@pytest.mark.parametrize("call", [fwd, bwd])
def test_residual_norm_refuses_a_branch(call):
    refused(call(rows=-1), "rows")
    refused(call(f=0), "rows of 0")
    refused(call(rows=1 << 30), "2^30")
    refused(call(rows=(1 << 31) - 1), "2^30")
    refused(call(f=(1 << 24) + 1), "2^24")
    refused(call(hd=gn.F16), "dtype")
    refused(call(hd=gn.F32, xd=gn.BF16), "dtype")
    refused(call(branch(post=3)), "kind")
    refused(call(branch(pre=-1)), "kind")
    refused(call(branch(post_w=BASE + 10 * MB)), "without their norm")
    refused(call(branch(pre=1)), "without their norm")
    refused(call(branch(gate=BASE + 10 * MB)), "gate and gates")
    refused(call(branch(gates=2)), "gate and gates")
    refused(call(branch(gate=BASE + 10 * MB, gates=-1)), "gate and gates")
    refused(call(branch(gate=BASE + 10 * MB, gates=4)), "multiple")
    refused(call(branch(p=1.0)), "p must be")
    refused(call(branch(p=float("nan"))), "p must be")
    refused(call(branch(p=0.5, rng=gn.Rng(0, 0, 0, 4))), "step_dev")
    refused(call(h=None), "null")
    refused(call(h=H + 1), "aligned")
    refused(call(branch(pre_w=BASE + 8 * MB + 1)), "aligned")
    refused(call(y=Y + 2), "aligned")


def test_residual_norm_refuses_outputs():
    refused(fwd(z=None), "z goes with")
    refused(fwd(branch(pre=0, pre_w=None, pre_b=None)), "z goes with")
    refused(fwd(x=None), "null")
    refused(fwd(y=X + 4), "share memory")
    refused(fwd(z=H), "share memory")
    refused(fwd(y=H), "share memory")
    refused(fwd(y=BASE + 8 * MB), "share memory")
    refused(fwd(branch(p=0.5, rng=gn.Rng(0, 0, 0, Y))), "share memory")
    refused(bwd(dz=DZ, b=branch(pre=0, pre_w=None, pre_b=None)), "dz goes with")
    refused(bwd(dy=None, dz=None), "neither")
    refused(bwd(y=None), "null")
    refused(bwd(dx=DY + 4), "share memory")
    refused(bwd(dh=DZ), "share memory")
    refused(bwd(dx=Y), "share memory")
    refused(bwd(g=gn.BranchGrads(G, None, None, None, None)), "without its parameter")
    refused(bwd(g=gn.BranchGrads(None, G, None, None, None)), "without its parameter")
    refused(bwd(g=gn.BranchGrads(None, None, None, G + 2, None)), "aligned")
    refused(bwd(g=gn.BranchGrads(None, None, None, G, G + 4)), "share memory")
    refused(bwd(g=gn.BranchGrads(None, None, None, G, WS + 64)), "share memory")
    need = gn.residual_norm_workspace_bytes(R, F)
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=WS + 8)):
        refused(bwd(g=gn.BranchGrads(None, None, None, G, None), **kw), "workspace", -3)
    refused(bwd(f=8200, rows=2, ws=None), "workspace", -3)  # wide rows need theirs with no gradient too


def test_workspace_query_of_refused_sizes():
    q = gn.lib().gn_residual_norm_workspace_bytes
    assert q(0, 8, 0) == q(4, 0, 0) == q(4, (1 << 24) + 1, 0) == q(4, 8, 3) == q(4, 8, -1) == q(1 << 30, 1, 0) == 0
    assert q(4, 8, 2) > 0


def test_no_rows():
    assert fwd(rows=0) == 0 and bwd(rows=0) == 0
