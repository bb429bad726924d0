"""Dropout, ResidualNorm and LinearAct as nodes of the tape, and the decoder that uses them: forward, tape backward, graph
replay, training steps.

Tolerances: a node's gradients are the direct call's, bit for bit; the decoder's are compared with fp32 torch
autograd of the same bf16-stored forward at the 2e-2 of the other decoder tests (normwise: a gradient passes some
ten bf16 roundings of 2^-8 each, in sums that cancel)."""
import math

import numpy as np
import pytest

from conftest import rel_err

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


@pytest.fixture(scope="module")
def env(gpu):
    import gn_bwd
    import grilly_bridge as gb
    import grilly_core
    dev = grilly_core.Device(0)
    gb.attach_torch_stream(dev)
    return grilly_core, gb, dev, gn_bwd


def rand(seed, *shape, dtype=BF, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def grad(gb, dev, tape, t, dtype=None):
    gid = tape.get_grad_buffer(t.data_ptr())
    assert gid != 0, "no gradient recorded"
    return gb.download(dev, gid, t.shape, gb.dtype_code(t) if dtype is None else dtype)


def host(t):
    return t.float().cpu().numpy()


def same(gb, dev, tape, t, want, dtype=None):
    np.testing.assert_array_equal(grad(gb, dev, tape, t, dtype), host(want))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_dropout_node(env, dtype):
    gc, gb, dev, gn = env
    x, dy = rand(1, 7, 33, dtype=dtype), rand(2, 7, 33, dtype=dtype)
    step = torch.tensor([5], device=DEV)
    y = gn.dropout_fwd(x, 0.3, 9, 4, step)
    for at, saved in ((0, [step.data_ptr()]), (5, [])):
        tape = gb.create_tape_context(dev)
        tape.begin()
        n = tape.record_op(gc.OpType.Dropout, [gb.tref(x, True)], [gb.tref(y)], gb.dropout_params(0.3, 9, 4, at))
        tape.save_for_backward(n, saved)
        tape.backward(n, dy.data_ptr())
        same(gb, dev, tape, x, gn.dropout_bwd(dy, 0.3, 9, 4, 5))
        tape.end()


@pytest.mark.parametrize("x_dtype,dtype", [(F32, BF), (BF, BF), (F32, F32)])
@pytest.mark.parametrize("ends", ["y", "z", "both"])
def test_residual_norm_node(env, x_dtype, dtype, ends):
    """With consumers of y, of z or of both behind it: Reshape nodes into two parts of a sum."""
    gc, gb, dev, gn = env
    rows, C = 12, 96
    h, x = rand(1, rows, C, dtype=dtype), rand(2, rows, C, dtype=x_dtype)
    w = [1 + rand(3, C, dtype=dtype, std=0.1), rand(4, C, dtype=dtype), 1 + rand(5, C, dtype=dtype, std=0.1), rand(6, C, dtype=dtype)]
    gate = rand(7, 3, C, dtype=dtype)
    kw = dict(post="layer", post_w=w[0], post_b=w[1], pre="layer", pre_w=w[2], pre_b=w[3], gate=gate, scale=0.5, res_scale=1.5,
              p=0.2, seed=3, stream=2, step=1)
    y, z = gn.residual_norm_fwd(h, x, **kw)
    dy, dz = rand(8, rows, C, dtype=x_dtype), rand(9, rows, C, dtype=dtype)
    want = gn.residual_norm_bwd(dy if ends != "z" else None, dz if ends != "y" else None, h, y, **kw)
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(op.ResidualNorm, [t(h, True), t(x, True)], [t(y), t(z)],
                       gb.residual_norm_params("layer", "layer", 3, 0.5, 1.5, 0.2, 3, 2, 1))
    tape.save_for_backward(n, [v.data_ptr() for v in w] + [gate.data_ptr()])
    if ends == "y":
        tape.backward(n, dy.data_ptr())  # as the root
    elif ends == "z":
        out = torch.empty_like(z)
        tape.backward(tape.record_op(op.Reshape, [t(z, True)], [t(out)]), dz.data_ptr())
    else:
        # z's gradient from a product with a constant, y's from the root, which both reach through one loss tensor
        one = torch.ones_like(z)
        mix = torch.empty_like(z)
        tape.record_op(op.Mul, [t(z, True), t(one)], [t(mix)])
        if x_dtype is dtype:
            out = torch.empty_like(y)
            want = gn.residual_norm_bwd(dy, dy, h, y, **kw)
            tape.backward(tape.record_op(op.Add, [t(y, True), t(mix, True)], [t(out)]), dy.data_ptr())
        else:
            out = torch.empty_like(y)
            want = gn.residual_norm_bwd(dy, dy.to(dtype), h, y, **kw)
            tape.backward(tape.record_op(op.Add, [t(y, True), t(mix, True)], [t(out)]), dy.data_ptr())
    same(gb, dev, tape, h, want[0])
    same(gb, dev, tape, x, want[1])
    for v, g in zip([gate] + w[:2], want[2:5]):
        same(gb, dev, tape, v, g, gb.DTYPE_F32)
    if ends != "y":
        for v, g in zip(w[2:], want[5:]):
            same(gb, dev, tape, v, g, gb.DTYPE_F32)
    tape.end()


def test_residual_norm_node_in_place(env):
    """The stream updated in place by two blocks: its id then holds the gradient of the version before both."""
    gc, gb, dev, gn = env
    rows, C = 10, 64
    x0 = rand(1, rows, C, dtype=F32)
    hs = [rand(2 + i, rows, C) for i in range(2)]
    w = 1 + rand(5, C, std=0.1)
    kw = dict(pre="rms", pre_w=w)
    # what two calls out of place give
    y1, z1 = gn.residual_norm_fwd(hs[0], x0, **kw)
    y2, z2 = gn.residual_norm_fwd(hs[1], y1, **kw)
    dy = rand(9, rows, C, dtype=F32)
    b2 = gn.residual_norm_bwd(dy, None, hs[1], y2, **kw)
    b1 = gn.residual_norm_bwd(b2[1], None, hs[0], y1, **kw)
    # the tape's backward reads y where pre has a gradient only, so that in place it needs no copy of y1 here
    x = x0.clone()
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.begin()
    for h in hs:
        n = tape.record_op(op.ResidualNorm, [t(h, True), t(x, True)], [t(x), t(z1)], gb.residual_norm_params(pre="rms"))
        tape.save_for_backward(n, [0, 0, w.data_ptr()])
    tape.backward(n, dy.data_ptr())
    same(gb, dev, tape, x, b1[1])
    same(gb, dev, tape, hs[0], b1[0])
    same(gb, dev, tape, hs[1], b2[0])
    tape.end()


@pytest.mark.parametrize("dtype,res", [(BF, None), (BF, F32), (BF, BF), (F32, None), (F32, F32)])
@pytest.mark.parametrize("act", ["none", "silu", "tanh"])
def test_linear_act_node(env, act, dtype, res):
    gc, gb, dev, gn = env
    M, N, K = 40, 64, 96
    X, W, b = rand(1, M, K, dtype=dtype), rand(2, N, K, dtype=dtype, std=0.1), rand(3, N, dtype=dtype)
    R = None if res is None else rand(4, M, N, dtype=res)
    Y, pre = gn.linear_act_fwd(X, W, b, act=act, residual=R, need_pre=True)
    dY = rand(5, M, N, dtype=Y.dtype)
    up = dY.to(dtype)
    dv = up if act == "none" else gn.act_bwd(act, up, pre)
    dX, dW, db = gn.linear_bwd(dv, X, W)
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(op.LinearAct, [t(X, True)] + ([] if R is None else [t(R, True)]), [t(Y)], gb.linear_act_params(act))
    tape.save_for_backward(n, [W.data_ptr(), b.data_ptr(), 0 if act == "none" else pre.data_ptr()])
    tape.backward(n, dY.data_ptr())
    same(gb, dev, tape, X, dX)
    same(gb, dev, tape, W, dW, gb.DTYPE_F32)
    same(gb, dev, tape, b, db, gb.DTYPE_F32)
    if R is not None:
        same(gb, dev, tape, R, dY)
    tape.end()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_tensor_as_both_inputs(env, dtype):
    """The residual that is the product's or the block's own input: one gradient, the sum of both (its terms rounded once
    each, and the sum: within a step of the terms' magnitudes)."""
    gc, gb, dev, gn = env
    M, K = 24, 64
    X, W, w = rand(1, M, K, dtype=dtype), rand(2, K, K, dtype=dtype, std=0.1), 1 + rand(3, K, dtype=dtype, std=0.1)
    op, t = gc.OpType, gb.tref
    dY = rand(5, M, K, dtype=dtype)
    Y, pre = gn.linear_act_fwd(X, W, act="silu", residual=X, need_pre=True)
    y, z = gn.residual_norm_fwd(X, X, post="layer", pre="rms", pre_w=w, p=0.2, seed=4)
    product = gn.linear_bwd(gn.act_bwd("silu", dY, pre), X, W)[0]
    dh, dx = gn.residual_norm_bwd(dY, None, X, y, post="layer", pre="rms", pre_w=w, p=0.2, seed=4)[:2]
    for node, inputs, outputs, params, saved, terms in (
            (op.LinearAct, [t(X, True), t(X, True)], [t(Y)], gb.linear_act_params("silu"), [W.data_ptr(), 0, pre.data_ptr()], (product, dY)),
            (op.ResidualNorm, [t(X, True), t(X, True)], [t(y), t(z)], gb.residual_norm_params(post="layer", pre="rms", p=0.2, seed=4),
             [0, 0, w.data_ptr()], (dh, dx))):
        tape = gb.create_tape_context(dev)
        tape.begin()
        n = tape.record_op(node, inputs, outputs, params)
        tape.save_for_backward(n, saved)
        tape.backward(n, dY.data_ptr())
        got, (a, b) = grad(gb, dev, tape, X).astype(np.float64), (host(v).astype(np.float64) for v in terms)
        assert (np.abs(got - a - b) <= torch.finfo(dtype).eps * (np.abs(a) + np.abs(b))).all()
        tape.end()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("behind", ["Linear", "LinearAct"])
@pytest.mark.parametrize("fused", [False, True])
def test_two_layers(env, dtype, behind, fused):
    """The activation's gradient in the product of the layer behind it, where that is asked for."""
    gc, gb, dev, gn = env
    M, d, ff = 72, 64, 136
    X, W1, b1 = rand(1, M, d, dtype=dtype), rand(2, ff, d, dtype=dtype, std=0.1), rand(3, ff, dtype=dtype)
    W2, b2 = rand(4, d, ff, dtype=dtype, std=0.1), rand(5, d, dtype=dtype)
    A, pre = gn.linear_act_fwd(X, W1, b1, act="gelu_tanh", need_pre=True)
    Y = gn.linear_act_fwd(A, W2, b2)
    dY = rand(6, M, d, dtype=dtype)
    if fused:
        dP, dW2, db2 = gn.act_linear_bwd("gelu_tanh", dY, pre, A, W2)
    else:
        dA, dW2, db2 = gn.linear_bwd(dY, A, W2)
        dP = gn.act_bwd("gelu_tanh", dA, pre)
    dX, dW1, db1 = gn.linear_bwd(dP, X, W1)
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(fused)
    tape.begin()
    n = tape.record_op(op.LinearAct, [t(X, True)], [t(A)], gb.linear_act_params("gelu_tanh"))
    tape.save_for_backward(n, [W1.data_ptr(), b1.data_ptr(), pre.data_ptr()])
    n = tape.record_op(getattr(op, behind), [t(A, True)], [t(Y)])
    tape.save_for_backward(n, [W2.data_ptr(), b2.data_ptr()])
    tape.backward(n, dY.data_ptr())
    same(gb, dev, tape, X, dX)
    for v, g in ((W1, dW1), (b1, db1), (W2, dW2), (b2, db2)):
        same(gb, dev, tape, v, g, gb.DTYPE_F32)
    assert (tape.get_grad_buffer(A.data_ptr()) == 0) == fused
    tape.end()


def test_activation_with_two_consumers_is_not_fused(env):
    gc, gb, dev, gn = env
    M, d = 24, 64
    X, W1, W2, W3 = rand(1, M, d), rand(2, d, d, std=0.1), rand(3, d, d, std=0.1), rand(4, d, d, std=0.1)
    A, pre = gn.linear_act_fwd(X, W1, act="silu", need_pre=True)
    Y, Z, S = (torch.empty_like(A) for _ in range(3))
    dY = rand(5, M, d)
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(True)
    tape.begin()
    n = tape.record_op(op.LinearAct, [t(X, True)], [t(A)], gb.linear_act_params("silu"))
    tape.save_for_backward(n, [W1.data_ptr(), 0, pre.data_ptr()])
    for w, o in ((W2, Y), (W3, Z)):
        n = tape.record_op(op.Linear, [t(A, True)], [t(o)])
        tape.save_for_backward(n, [w.data_ptr()])
    tape.backward(tape.record_op(op.Add, [t(Y, True), t(Z, True)], [t(S)]), dY.data_ptr())
    dA = gn.linear_bwd(dY, A, W3)[0] + gn.linear_bwd(dY, A, W2)[0]
    same(gb, dev, tape, A, dA)
    same(gb, dev, tape, X, gn.linear_bwd(gn.act_bwd("silu", dA, pre), X, W1)[0])
    tape.end()


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_activation_that_is_its_consumers_residual_is_not_fused(env, dtype, fused):
    gc, gb, dev, gn = env
    M, d = 24, 64
    X, W1, W2 = rand(1, M, d, dtype=dtype), rand(2, d, d, dtype=dtype, std=0.1), rand(3, d, d, dtype=dtype, std=0.1)
    A, pre = gn.linear_act_fwd(X, W1, act="silu", need_pre=True)
    Y = gn.linear_act_fwd(A, W2, residual=A)
    dY = rand(5, M, d, dtype=dtype)
    op, t = gc.OpType, gb.tref
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(fused)
    tape.begin()
    n = tape.record_op(op.LinearAct, [t(X, True)], [t(A)], gb.linear_act_params("silu"))
    tape.save_for_backward(n, [W1.data_ptr(), 0, pre.data_ptr()])
    n = tape.record_op(op.LinearAct, [t(A, True), t(A, True)], [t(Y)])
    tape.save_for_backward(n, [W2.data_ptr()])
    tape.backward(n, dY.data_ptr())
    dA = gn.linear_bwd(dY, A, W2)[0] + dY
    same(gb, dev, tape, A, dA)
    same(gb, dev, tape, X, gn.linear_bwd(gn.act_bwd("silu", dA, pre), X, W1)[0])
    tape.end()


def test_nodes_refuse(env):
    gc, gb, dev, gn = env
    x, y = rand(1, 4, 8), rand(2, 4, 8)
    w = rand(3, 8, 8)

    def go(op, params, saved, match):
        tape = gb.create_tape_context(dev)
        tape.begin()
        n = tape.record_op(op, [gb.tref(x, True)], [gb.tref(y)], params)
        tape.save_for_backward(n, saved)
        with pytest.raises((ValueError, RuntimeError), match=match):
            tape.backward(n, x.data_ptr())
        tape.end()

    op = gc.OpType
    go(op.Dropout, b"", [], "must hold p")
    go(op.Dropout, gb.dropout_params(1.0, 0), [], "p must be")
    go(op.LinearAct, gb.linear_act_params("silu"), [0], "must hold W")
    go(op.LinearAct, gb.linear_act_params("silu"), [w.data_ptr()], "must hold P")


# ---- the decoder -------------------------------------------------------------------------
def factors(p, n, seed, stream, step):
    """The masks' factors through dropout_fwd, which tests of its own hold to its definition."""
    import gn_bwd
    return gn_bwd.dropout_fwd(torch.ones(n, device=DEV), p, seed, stream, step)


def reference(m):
    """fp32 torch autograd of the decoder, rounding to bf16 where the GPU run stores (straight through)."""
    rb = lambda t: t + (t.bfloat16().float() - t).detach()
    leaf = lambda t: t.detach().float().clone().requires_grad_(True)
    B, S, H, d, T = m.B, m.S, m.H, m.d, m.T
    E = leaf(m.E)
    params = [{k: leaf(v) for k, v in p.items()} for p in m.layers]
    lnf_g, lnf_b = leaf(m.lnf_g), leaf(m.lnf_b)
    step = int(m.step)
    drop = lambda t, place: t * factors(m.p, T * d, m.seed, place, step).view(T, d) if m.p else t  # noqa: E731

    def ln(x, g, b):
        mu = x.mean(-1, keepdim=True)
        return rb((x - mu) * torch.rsqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5) * g + b)

    def gelu(u):
        return 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3)))

    mask = torch.triu(torch.ones(S, S, dtype=torch.bool, device=DEV), 1)
    x = drop(E[m.ids.long()], 0)
    for i, p in enumerate(params):
        qkv = rb(ln(x, p["ln1_g"], p["ln1_b"]) @ p["Wqkv"].t() + p["bqkv"]).view(B, S, 3, H, d // H)
        q, k, v = qkv.permute(2, 0, 3, 1, 4)
        sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d // H)
        o = torch.matmul(torch.softmax(sc.masked_fill(mask, float("-inf")), -1), v)
        ao = rb(o.permute(0, 2, 1, 3).reshape(T, d)) @ p["Wo"].t() + p["bo"]
        x2 = x + (ao if m.fused_linear else drop(rb(ao), 2 * i + 1))
        n2 = ln(x2, p["ln2_g"], p["ln2_b"])
        up = n2 @ p["Wu"].t() + p["bu"]
        h = rb(gelu(up)) if m.ffn == "gelu" else rb(rb(n2 @ p["Wg"].t() + p["bg"]) * gelu(rb(up)))
        f = h @ p["Wd"].t() + p["bd"]
        x = x2 + (f if m.fused_linear else drop(rb(f), 2 * i + 2))
    logits = ln(x, lnf_g, lnf_b) @ E.t()
    torch.nn.functional.cross_entropy(logits, m.tgt.long()).backward()
    return E, params, lnf_g, lnf_b


OPTIONS = [dict(residual_norm=True), dict(residual_norm=True, dropout=0.2), dict(fused_linear=True),
           dict(fused_linear=True, ffn="gelu"), dict(residual_norm=True, dropout=0.1, ffn="gelu", fused_loss=True), dict(ffn="gelu")]


def model(seed, **options):
    import decoder_tape
    m = decoder_tape.Decoder(layers=2, d=128, heads=2, ff=256, vocab=301, batch=2, seq=129, seed=seed, **options)
    m.step.fill_(3)
    for i, p in enumerate(m.layers):
        for j, k in enumerate(("ln1_g", "ln2_g")):
            p[k].copy_(1 + rand(seed + 10 * i + j, *p[k].shape, dtype=F32, std=0.2))
        for j, k in enumerate(("ln1_b", "ln2_b", "bqkv", "bo", "bg", "bu", "bd")):
            p[k].copy_(rand(seed + 10 * i + j + 3, *p[k].shape, dtype=F32, std=0.05))
    return m


def keys(m):
    return ("Wqkv", "bqkv", "Wo", "bo", "ln1_g", "ln1_b", "ln2_g", "ln2_b", "Wu", "bu", "Wd", "bd") + (("Wg", "bg") if m.ffn == "geglu" else ())


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(f"{k}={v}" for k, v in o.items()))
def test_decoder(env, options):
    gc, gb, dev, gn = env
    m = model(7, **options)
    m.forward()
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(True)
    tape.begin()
    tape.backward(m.record(tape), 0)
    E, params, lnf_g, lnf_b = reference(m)
    tensors = [("E", m.E, E), ("lnf_g", m.lnf_g, lnf_g), ("lnf_b", m.lnf_b, lnf_b)]
    for i, (p, r) in enumerate(zip(m.layers, params)):
        tensors += [(f"{k}{i}", p[k], r[k]) for k in keys(m)]
    errs = {k: rel_err(grad(gb, dev, tape, t, gb.DTYPE_F32), r.grad.cpu().numpy()) for k, t, r in tensors}
    tape.end()
    bad = {k: v for k, v in errs.items() if not v < 2e-2}
    assert not bad, f"relative errors above 2e-2: {bad} (all: {errs})"


@pytest.mark.parametrize("options", [OPTIONS[4], OPTIONS[3]], ids=["residual_norm", "fused_linear"])
def test_decoder_backward_replayed(env, options):
    """Captured once into a graph of kernel nodes only, while an eager pass of the same tensors lives; replays equal the eager
    backward (the tied table, whose embedding part sums fp32 atomics, within 1e-6)."""
    gc, gb, dev, gn = env
    m = model(8, **options)
    m.forward()
    tensors = {"E": m.E, "lnf_g": m.lnf_g}
    for i, p in enumerate(m.layers):
        tensors.update({f"{k}{i}": p[k] for k in keys(m)})
    tape = gb.create_tape_context(dev)
    tape.set_glu_epilogue(True)
    tape.begin()
    graph = gc.OpGraph()
    graph.capture_backward(tape, m.record(tape), 0)
    tape.end()
    assert graph.node_counts()["memset"] == 0 and graph.node_counts()["memcpy"] == 0
    for rep in range(4):
        if rep:
            m.step.fill_(3 + rep)
            m.forward()  # new activations are new tensors: the graph's stay, and so the masks must be those of its forward
            m.step.fill_(3)
        torch.cuda.synchronize()
        graph.execute(dev)
        torch.cuda.synchronize()
        if rep == 0:
            eager = gb.create_tape_context(dev)
            eager.set_glu_epilogue(True)
            eager.begin()
            eager.backward(m.record(eager), 0)
            want = {k: grad(gb, dev, eager, t, gb.DTYPE_F32) for k, t in tensors.items()}
            eager.end()
            keep = m.acts, m.x0, getattr(m, "x0d", None), m.nf, getattr(m, "logits", None)  # noqa: F841
            keep += (getattr(m, "lse", None), getattr(m, "mf", None), getattr(m, "rf", None), getattr(m, "row_loss", None))
        for k, t in tensors.items():
            a = gb.download(dev, graph.get_grad_buffer(t.data_ptr()), t.shape, gb.DTYPE_F32)
            if k == "E":
                assert rel_err(a, want[k]) < 1e-6
            else:
                np.testing.assert_array_equal(a, want[k], err_msg=f"replay {rep}: {k}")
    graph.clear()


@pytest.mark.parametrize("options", [OPTIONS[4], OPTIONS[3]], ids=["residual_norm", "fused_linear"])
def test_training_steps(env, options):
    """Three steps of forward, tape backward and AdamW, the masks' step counted on: every weight with a gradient moves, and
    stays finite."""
    gc, gb, dev, gn = env
    m = model(10, **options)
    weights = [m.E, m.lnf_g] + [p[k] for p in m.layers for k in keys(m)]
    before = [w.clone() for w in weights]
    opt = gb.AdamW(weights, lr=1e-2)
    tape = gb.create_tape_context(dev)
    for _ in range(3):
        m.forward()
        tape.begin()
        tape.backward(m.record(tape), 0)
        assert opt.step(tape) == len(weights)
        tape.end()
        m.step += 1
    torch.cuda.synchronize()
    for w, b in zip(weights, before):
        assert bool(torch.isfinite(w).all()) and not torch.equal(w, b)
